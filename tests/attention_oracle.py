"""The attention operators' definitions in 64 bits, with the bounds that the kernels' arithmetic keeps to.

A value that is stored in type t is off by at most half a step, u(t) = finfo(t).eps / 2 relative to it (fp16: plus 2^-25 where
it falls below the normal numbers).  Probabilities and score gradients enter the second matrix products in the inputs' type:
one more u(t) on every term of those sums (fp32: none).  Sums run in fp32: a sum of n terms is off by at most n 2^-24 of the
sum of their magnitudes, which also bounds the fp32 score's error, and through exp the probabilities' relative error."""
import math

import torch

BLOCK = 64
F32 = 2.0 ** -24


def unit(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 0.0


def live(b, n, arr):
    return [n] * b if arr is None else [max(0, min(n, int(x))) for x in arr]


def means(k, n_arr=None):
    """(B,nb,Hk,D) float64"""
    b, n, hk, d = k.shape
    nb = -(-n // BLOCK)
    out = torch.zeros((b, nb, hk, d), dtype=torch.float64, device=k.device)
    for e, ln in enumerate(live(b, n, n_arr)):
        for j in range(-(-ln // BLOCK)):
            out[e, j] = k[e, j * BLOCK:min(ln, (j + 1) * BLOCK)].double().mean(dim=0)
    return out


def select(q, mean, keys, count, n_arr=None, m_arr=None, causal=False):
    b, m, hq, d = q.shape
    hk, nb = mean.size(2), mean.size(1)
    out = torch.full((b, m, hk, count), -1, dtype=torch.int32)
    for e, (ln, lm) in enumerate(zip(live(b, keys, n_arr), live(b, m, m_arr))):
        total = q[e].double().view(m, hk, hq // hk, d).sum(dim=2)
        score = torch.einsum("mhd,bhd->hmb", total, mean[e].double()).cpu()
        score = torch.where(score.isnan(), torch.full_like(score, -math.inf), score)
        for i in range(lm):
            p = ln - lm + i
            end = -(-ln // BLOCK) if not causal else p // BLOCK + 1 if p >= 0 else 0
            for h in range(hk):
                row = score[h, i, :end].clone()
                if causal and end:
                    row[end - 1] = math.inf
                best = torch.sort(row, descending=True, stable=True)[1][:count].sort()[0]
                out[e, i, h, :best.numel()] = best.int()
    return out


def seen(b, m, n, hk, blocks, n_arr=None, m_arr=None, causal=False):
    """(B,Hk,M,N) bool: which keys a query sees."""
    dev = blocks.device
    nb = -(-n // BLOCK)
    hit = torch.zeros((b, hk, m, nb + 1), dtype=torch.bool, device=dev)
    idx = blocks.long().transpose(1, 2)
    idx = torch.where((idx < 0) | (idx >= nb), torch.full_like(idx, nb), idx)
    hit.scatter_(3, idx, True)
    key = torch.arange(n, device=dev)
    see = hit[..., :nb][..., key // BLOCK] if n else torch.zeros((b, hk, m, 0), dtype=torch.bool, device=dev)
    row = torch.arange(m, device=dev)
    for e, (ln, lm) in enumerate(zip(live(b, n, n_arr), live(b, m, m_arr))):
        see[e] &= (key < ln) & (row < lm)[:, None]
        if causal:
            see[e] &= key <= (row + ln - lm)[:, None]
    return see


def attention(q, k, v, blocks, scale=None, n_arr=None, m_arr=None, causal=False, go=None):
    """-> dict of float64 results o[, dq, dk, dv] and the bound of each (t_o, ...), all (B, rows, heads, D)."""
    dt = q.dtype
    b, m, hq, d = q.shape
    n, hk = k.size(1), k.size(2)
    g = hq // hk
    scale = d ** -0.5 if scale is None else scale
    see = seen(b, m, n, hk, blocks, n_arr, m_arr, causal)
    some = see.any(dim=2).any(dim=1)                                      # rows that nobody sees do not matter
    clean = lambda t, keep: torch.where(keep[:, :, None, None], t.detach().double(), torch.zeros((), dtype=torch.float64, device=t.device))  # noqa: E731
    kf, vf = clean(k, some), clean(v, some)
    qf = clean(q, see.any(dim=3).any(dim=1))
    qf, kf, vf = (t.transpose(1, 2) for t in (qf, kf, vf))
    kf, vf = kf.repeat_interleave(g, dim=1), vf.repeat_interleave(g, dim=1)
    see = see.repeat_interleave(g, dim=1)
    x = scale * (qf @ kf.transpose(2, 3))
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    top = x.amax(dim=3, keepdim=True) if n else torch.zeros((b, hq, m, 1), dtype=torch.float64, device=q.device)
    p = torch.exp(x - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = p.sum(dim=3, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = p @ vf
    terms = see.sum(dim=3, keepdim=True).double()
    # fp32 scores: d + 3 roundings on the sum of magnitudes (the scale, its product, the base-2 exponent); exp and its base
    # turn an absolute error into a relative one, the denominator has the same
    xe = torch.where(see, scale * (qf.abs() @ kf.abs().transpose(2, 3)), torch.zeros_like(x))
    xe = (xe.amax(dim=3, keepdim=True) if n else torch.zeros_like(top)) * (d + 8) * F32
    pe = 2 * xe + (terms + 16) * F32                                       # relative error of a probability
    # (16-bit types: the denominator adds up the rounded probabilities, each w off, so it is w off itself: o is off by w |o|
    # more, and the probabilities that the backward pass forms with it by w)
    u, w = unit(dt), unit(dt) if dt != torch.float32 else 0.0
    mag = p @ vf.abs()
    t_o = (u + w) * o.abs() + (w + pe + terms * F32) * mag + tiny(dt) * (1 + (see.double() @ vf.abs()))
    back = lambda t: t.transpose(1, 2)                                     # noqa: E731
    pe = pe + w
    out = dict(o=back(o), t_o=1.05 * back(t_o) + 1e-30)
    if go is None:
        return out
    gf = clean(go, see.any(dim=3).any(dim=1)).transpose(1, 2)
    dp = gf @ vf.transpose(2, 3)
    delta = (gf * o).sum(dim=3, keepdim=True)
    ds = torch.where(see, p * (dp - delta), torch.zeros_like(p))
    group = lambda t: t.view(b, hk, g, n, d).sum(dim=2)                    # noqa: E731
    dq, dk, dv = scale * (ds @ kf), group(scale * (ds.transpose(2, 3) @ qf)), group(p.transpose(2, 3) @ gf)
    # do . v in fp32; do . o with the rounded o
    edp = (gf.abs() @ vf.abs().transpose(2, 3)) * (d + 2) * F32
    ede = (gf.abs() * t_o).sum(dim=3, keepdim=True) + (d + 2) * F32 * (gf * o).abs().sum(dim=3, keepdim=True)
    big = gf.abs().amax(dim=3, keepdim=True)
    e = torch.where(see, ds.abs() * (w + pe) + p * (edp + ede) + 2 * tiny(dt) * big, torch.zeros_like(p))
    rows = see.sum(dim=2).unsqueeze(3).double().amax(dim=2, keepdim=True) * g if n else torch.zeros((b, hq, 1, 1), dtype=torch.float64, device=q.device)
    t_dq = u * dq.abs() + scale * ((e + ds.abs() * terms * F32) @ kf.abs()) + tiny(dt)
    t_dk = u * dk.abs() + group(scale * ((e + ds.abs() * rows * F32).transpose(2, 3) @ qf.abs())) + tiny(dt)
    t_dv = u * dv.abs() + group(((p * (w + pe) + p * rows * F32 + see * tiny(dt)).transpose(2, 3)) @ gf.abs()) + tiny(dt)
    out.update(dq=back(dq), dk=back(dk), dv=back(dv), t_dq=1.05 * back(t_dq) + 1e-30, t_dk=1.05 * back(t_dk) + 1e-30,
               t_dv=1.05 * back(t_dv) + 1e-30)
    return out


def norm_rotate(x, w, position, freq, eps=1e-6, interleaved=False, g=None):
    """One side of norm_rotate in 64 bits: y and its bound; with g (gradient of y): dx, dw and theirs.  x (B,N,H,D)."""
    b, n, h, d = x.shape
    dt = x.dtype
    p = position.double()
    p = p.unsqueeze(2) if p.dim() == 2 else p
    a = (p.unsqueeze(3) * freq.double()).flatten(2).unsqueeze(2)           # (B,N,1,R)
    r = a.size(3)
    at = torch.arange(r, device=x.device)
    one, two = (2 * at, 2 * at + 1) if interleaved else (at, at + r)
    c, s = torch.cos(a), torch.sin(a)

    def turn(t, sign):
        y = t.clone()
        y[..., one] = t[..., one] * c - sign * t[..., two] * s
        y[..., two] = sign * t[..., one] * s + t[..., two] * c
        return y

    def both(t):                                                           # |one| + |two| in both places
        y = t.abs().clone()
        y[..., one] = t[..., one].abs() + t[..., two].abs()
        y[..., two] = y[..., one]
        return y

    xf = x.detach().double()
    inv = 1 / torch.sqrt((xf * xf).mean(dim=3, keepdim=True) + eps)
    unit_x = xf * inv
    wf = torch.ones((d,), dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    y = unit_x * wf
    u = unit(dt)
    # mean and root: (d + 4) / 2 + 3 roundings relative; weights, products; sine and cosine within 4 roundings of 1
    rel = (d / 2 + 16) * F32
    out = dict(y=turn(y, 1.0), t_y=u * turn(y, 1.0).abs() + rel * both(y) + tiny(dt))
    if g is None:
        return out
    hb = turn(g.detach().double(), -1.0)
    mag = both(g.detach().double())
    gw = hb * wf
    dot = (gw * unit_x).mean(dim=3, keepdim=True)
    dx = inv * (gw - unit_x * dot)
    size = inv * (mag * wf.abs() + unit_x.abs() * (mag * wf.abs() * unit_x.abs()).mean(dim=3, keepdim=True))
    out.update(dx=dx, t_dx=u * dx.abs() + (2 * d + 48) * F32 * size + tiny(dt))
    if w is not None:
        dims = (0, 1) if w.dim() == 2 else (0, 1, 2)
        dw = (hb * unit_x).sum(dim=dims)
        rows = b * n * (1 if w.dim() == 2 else h)
        sizes = (mag * unit_x.abs()).sum(dim=dims)
        # a partial sum holds at most as many rows as there are; the partial sums are added in 64 bits
        out.update(dw=dw, t_dw=unit(w.dtype) * dw.abs() + (min(rows, 4096) + d / 2 + 32) * F32 * sizes + tiny(w.dtype))
    return out
