"""gpu: the attention operators at the ends of their types' range and of their interface: results against the plain form in
32 bits, scores, values and gradients that are very large or very small, values that are not finite in every gradient,
derivatives that are not offered, kept means, several threads.

Errors are measured against 64 bits.  The plain form computes in fp32 and rounds once; the kernels' 16-bit operands of the second
matrix products are two terms of the type, which hold 2^-17 (bf16) or 2^-22 (fp16) of a value: 2^-9 or less of what the last
rounding takes, so that the two errors differ by far less than the 5 % that the tests allow."""
import math
import threading

import pytest
import torch

import attention_oracle as orc64
from conftest import pkg

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, device=gen.device, generator=gen).to(dtype)


def _inputs(dev, b, m, n, hq, hk, d, count, dtype, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    q, k, v = _randn(gen, b, m, hq, d, dtype=dtype), _randn(gen, b, n, hk, d, dtype=dtype), _randn(gen, b, n, hk, d, dtype=dtype)
    go = _randn(gen, b, m, hq, d, dtype=dtype)
    nb = -(-n // 64)
    blocks = torch.rand((b, m, hk, nb), device=dev, generator=gen).sort(dim=3)[1][..., :count].sort(dim=3)[0].to(torch.int32)
    return q, k, v, go, blocks


def _formula(q, k, v, blocks, scale, causal, go, dtype):
    """o, dq, dk, dv by the formulas in `dtype`, not rounded."""
    b, m, hq, d = q.shape
    n, hk = k.size(1), k.size(2)
    g = hq // hk
    see = orc64.seen(b, m, n, hk, blocks, None, None, causal).repeat_interleave(g, dim=1)
    qf, kf, vf, gf = (t.detach().to(dtype).transpose(1, 2).contiguous() for t in (q, k, v, go))
    kf, vf = kf.repeat_interleave(g, dim=1), vf.repeat_interleave(g, dim=1)
    x = scale * (qf @ kf.transpose(2, 3).contiguous())
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    p = torch.exp(x - x.amax(dim=3, keepdim=True))
    p = p / p.sum(dim=3, keepdim=True)
    o = p @ vf
    ds = p * (gf @ vf.transpose(2, 3).contiguous() - (gf * o).sum(dim=3, keepdim=True))
    sums = [scale * (ds @ kf), scale * (ds.transpose(2, 3).contiguous() @ qf), p.transpose(2, 3).contiguous() @ gf]
    sums[1:] = [t.view(b, hk, g, n, d).sum(dim=2) for t in sums[1:]]
    return [t.transpose(1, 2) for t in [o] + sums]


def _error(got, want, where=None):
    """Root of the mean square of what is off, relative to the same of what is right."""
    got, want = got.detach().double(), want.double()
    if where is not None:
        got, want = got[where], want[where]
    return ((got - want).pow(2).mean().sqrt() / want.pow(2).mean().sqrt()).item()


def _run(ops, leaves, go, *args, **kw):
    leaves = [t.detach().clone().requires_grad_() for t in leaves]
    o = ops.block_attention(*leaves, *args, **kw)
    return (o.detach(),) + torch.autograd.grad(o, leaves, go)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("b,m,n,hq,hk,d,count,causal", [(2, 300, 1024, 4, 2, 64, 6, False), (1, 600, 600, 6, 2, 128, 4, True),
                                                        (3, 400, 700, 2, 2, 24, 3, False), (2, 3, 4000, 8, 2, 128, 16, False)])
def test_errors_of_16_bit_types_are_their_last_rounding(dev, b, m, n, hq, hk, d, count, causal, dtype):
    ops = pkg("network.operations")
    q, k, v, go, blocks = _inputs(dev, b, m, n, hq, hk, d, count, TYPES[dtype], 11)
    if causal:                                              # (every query sees something)
        blocks[..., 0] = 0
    scale = d ** -0.5
    want = _formula(q, k, v, blocks, scale, causal, go, torch.float64)
    plain = _formula(q, k, v, blocks, scale, causal, go, torch.float32)
    for name, x, y, z in zip(("o", "dq", "dk", "dv"), _run(ops, (q, k, v), go, blocks, causal=causal), plain, want):
        here, there = _error(x, z), _error(y.to(q.dtype), z)
        print("%s: %.3g, plain %.3g" % (name, here, there))
        assert here <= 1.05 * there, (name, here, there)
