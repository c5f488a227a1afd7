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


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("queries", [200, 2])
def test_scores_far_beyond_the_exponents_range(dev, dtype, queries):
    """Scores of up to 2^33 (fp16) and 2^87, all exact in fp32 and far apart: the largest key has all the weight, so the output is its
    value, dv the sum of the gradients of the rows that chose it, and ds, dq, dk are 0, all exactly."""
    ops = pkg("network.operations")
    gen = torch.Generator(device=dev).manual_seed(5)
    dt, n, d = TYPES[dtype], 128, 64
    big = 2.0 ** (13 if dt == torch.float16 else 40)
    pattern = torch.sign(_randn(gen, d))
    w = 1 + torch.randperm(n, device=dev, generator=gen).float() / 128
    side = torch.tensor([1.0, -1.0], device=dev).repeat(queries // 2)                           # odd rows want the smallest
    row = side * (1 + torch.arange(queries, device=dev) % 128 / 128)
    q = (big * row[:, None] * pattern).to(dt).view(1, queries, 1, d)
    k = (big * w[:, None] * pattern).to(dt).view(1, n, 1, d)
    v = torch.randint(-8, 9, (1, n, 1, d), device=dev, generator=gen).to(dt)
    go = torch.randint(-1, 2, (1, queries, 1, d), device=dev, generator=gen).to(dt)
    blocks = torch.tensor([0, 1], dtype=torch.int32, device=dev).expand(1, queries, 1, 2)
    o, dq, dk, dv = _run(ops, (q, k, v), go, blocks)
    best, worst = w.argmax(), w.argmin()
    assert torch.equal(o, torch.where((side > 0).view(1, -1, 1, 1), v[:, best:best + 1], v[:, worst:worst + 1]))
    want = torch.zeros_like(v)
    want[0, best], want[0, worst] = go[0, side > 0].sum(dim=0), go[0, side < 0].sum(dim=0)
    assert torch.equal(dv, want) and (dq == 0).all() and (dk == 0).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_gradients_of_scores_with_a_large_common_part(dev, dtype):
    """Scores of 2^20 + {0 .. 7}, exact in fp32: the probabilities are those of 0 .. 7.  A probability is off by the rounding of the
    exponent, of exp2 and of the sum, together below 2^-19, and by its two terms in the 16-bit types (2^-17): 2^-15 of the sum
    of magnitudes, and the last rounding."""
    ops = pkg("network.operations")
    gen = torch.Generator(device=dev).manual_seed(6)
    dt, n, m, d = TYPES[dtype], 256, 150, 32
    q, k = torch.zeros((1, m, 1, d), device=dev), torch.zeros((1, n, 1, d), device=dev)
    q[..., 0], k[..., 0] = 1024, 1024
    q[..., 1] = 1
    k[..., 1] = torch.randint(0, 8, (1, n, 1), device=dev, generator=gen).float()
    q, k = q.to(dt), k.to(dt)
    v, go = _randn(gen, 1, n, 1, d, dtype=dt), _randn(gen, 1, m, 1, d, dtype=dt)
    blocks = torch.arange(4, dtype=torch.int32, device=dev).expand(1, m, 1, 4)
    o, _, _, dv = _run(ops, (q, k, v), go, blocks, 1.0)
    p = torch.softmax(k[0, :, 0, 1].double(), dim=0)
    u = torch.finfo(dt).eps / 2
    for got, want, size in ((o, p @ v[0, :, 0].double(), p @ v[0, :, 0].double().abs()),
                            (dv, p[:, None] * go[0, :, 0].double().sum(dim=0), p[:, None] * go[0, :, 0].double().abs().sum(dim=0))):
        assert ((got[0, :, 0].double() - want).abs() <= u * want.abs() + 2.0 ** -15 * size + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_keys_and_values_that_are_not_numbers_in_the_gradients_of_keys(dev, dtype):
    """A key that is NaN: the rows that see it have no probabilities, so dk and dv of every key that one of them sees are not
    numbers, as whole rows.  A value that is NaN: the same for dk; dv does not depend on it.  All others have the bits of a
    call without them."""
    ops = pkg("network.operations")
    q, k, v, go, _ = _inputs(dev, 1, 128, 192, 2, 1, 64, 1, TYPES[dtype], 61)
    blocks = torch.zeros((1, 128, 1, 2), dtype=torch.int32, device=dev)
    blocks[:, ::2, :, 1] = 1
    blocks[:, 1::2, :, 1] = 2
    see = orc64.seen(1, 128, 192, 1, blocks, causal=True)[0, 0]
    _, _, dk2, dv2 = _run(ops, (q, k, v), go, blocks, causal=True)
    for bad in (70, 100, 150):
        hit = see[see[:, bad]].any(dim=0)
        assert hit.any() and not hit.all()
        kk = k.clone()
        kk[0, bad, 0, 3] = math.nan
        _, _, dk, dv = _run(ops, (q, kk, v), go, blocks, causal=True)
        assert dk[0, hit].isnan().all() and dv[0, hit].isnan().all()
        assert torch.equal(dk[0, ~hit], dk2[0, ~hit]) and torch.equal(dv[0, ~hit], dv2[0, ~hit])
        vv = v.clone()
        vv[0, bad, 0, 5] = math.nan
        _, _, dk, dv = _run(ops, (q, k, vv), go, blocks, causal=True)
        assert dk[0, hit].isnan().all() and torch.equal(dv, dv2)
        assert torch.equal(dk[0, ~hit], dk2[0, ~hit])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("queries", [130, 2])
def test_rows_whose_scores_are_all_minus_infinity(dev, dtype, queries):
    """Such a row is 0 and passes no gradient on to the keys and values it sees; its own gradient is 0 where the keys are finite
    (scores that overflow), not a number where they are not."""
    ops = pkg("network.operations")
    q, k, v, go, _ = _inputs(dev, 1, queries, 128, 2, 1, 64, 1, TYPES[dtype], 62)
    blocks = (torch.arange(queries, device=dev) % 2).to(torch.int32).view(1, -1, 1, 1)
    infinite = TYPES[dtype] == torch.float16
    q[..., 0] = 1000 if infinite else 1e25
    k[..., 0] = 0
    k[0, 64:, 0, 0] = -math.inf if infinite else -1e25
    o, dq, dk, dv = _run(ops, (q, k, v), go, blocks)
    assert (o[0, 1::2] == 0).all() and (dk[0, 64:] == 0).all() and (dv[0, 64:] == 0).all()
    assert dq[0, 1::2].isnan().all() if infinite else (dq[0, 1::2] == 0).all()
    keep = slice(0, None, 2)
    alone = _run(ops, (q[:, keep], k, v), go[:, keep], blocks[:, keep])
    assert torch.equal(o[:, keep], alone[0]) and torch.isfinite(dk[0, :64]).all() and torch.isfinite(dv[0, :64]).all()
    assert torch.isfinite(dq[:, keep]).all()


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-5])
def test_fp16_gradients_of_small_values(dev, size):
    """Values far below 1 (down to where the output itself is below fp16's normal numbers) and gradients of 256: score gradients
    small against |do|, results that are normal numbers."""
    ops = pkg("network.operations")
    q, k, v, go, blocks = _inputs(dev, 1, 260, 1024, 2, 1, 128, 16, torch.float16, 21)
    v, go = (size * v.float()).half(), 256 * go
    scale = 128 ** -0.5
    want = _formula(q, k, v, blocks, scale, False, go, torch.float64)
    plain = _formula(q, k, v, blocks, scale, False, go, torch.float32)
    got = _run(ops, (q, k, v), go, blocks)
    for i, name in ((1, "dq"), (2, "dk"), (3, "dv")):
        rows = want[i].shape[1]
        worst = max((_error(got[i][:, r], want[i][:, r]) / _error(plain[i][:, r].half(), want[i][:, r]) for r in range(rows)))
        here, there = _error(got[i], want[i]), _error(plain[i].half(), want[i])
        print("%s: %.3g, plain %.3g, worst row %.3g of the plain form's" % (name, here, there, worst))
        assert here <= 1.05 * there, (name, here, there)


def test_fp16_gradients_of_keys_with_little_weight(dev):
    """Every fourth key has e^-14 of the others' weight: its gradients are as exact, relative to them, as the others'."""
    ops = pkg("network.operations")
    q, k, v, go, blocks = _inputs(dev, 1, 300, 1024, 1, 1, 64, 16, torch.float16, 22)
    q[..., 0] = 4
    k[..., 0] = 0
    k[:, ::4, :, 0] = -28
    go = 256 * go
    want = _formula(q, k, v, blocks, 0.125, False, go, torch.float64)
    plain = _formula(q, k, v, blocks, 0.125, False, go, torch.float32)
    got = _run(ops, (q, k, v), go, blocks)
    few = torch.zeros((1, 1024), dtype=torch.bool, device=dev)
    few[:, ::4] = True
    for i, name in ((2, "dk"), (3, "dv")):
        here, there = _error(got[i], want[i], few), _error(plain[i].half(), want[i], few)
        print("%s: %.3g, plain %.3g" % (name, here, there))
        assert here <= 1.05 * there, (name, here, there)


@pytest.mark.parametrize("large", [60000.0, math.inf])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_a_large_gradient_leaves_unseeing_keys_alone(dev, dtype, large):
    """One query's output gradient is very large, or infinite, beside gradients of 1e-4: the keys that it does not see have the
    gradients they have without it, to the bit."""
    ops = pkg("network.operations")
    q, k, v, go, _ = _inputs(dev, 1, 256, 256, 2, 1, 64, 1, TYPES[dtype], 23)
    go = 1e-4 * go
    blocks = torch.arange(4, dtype=torch.int32, device=dev).expand(1, 256, 1, 4)
    for i in (20, 150):
        pair = [go.clone(), go.clone()]
        pair[0][0, i, 1] = large
        pair[1][0, i, 1] = 0
        _, dq, dk, dv = _run(ops, (q, k, v), pair[0], blocks, causal=True)
        _, dq2, dk2, dv2 = _run(ops, (q, k, v), pair[1], blocks, causal=True)
        assert torch.equal(dk[0, i + 1:], dk2[0, i + 1:]) and torch.equal(dv[0, i + 1:], dv2[0, i + 1:])
        others = torch.arange(256, device=dev) != i
        assert torch.equal(dq[0, others], dq2[0, others])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("queries", [70, 1])
def test_values_at_the_types_end(dev, dtype, queries):
    """A mean of values near the largest number of the type is near it, and no sum on the way to it leaves the range."""
    ops = pkg("network.operations")
    dt = TYPES[dtype]
    q, k, _, _, blocks = _inputs(dev, 1, queries, 2000, 2, 1, 64, 20, dt, 8)
    top = 65504.0 if dt == torch.float16 else 3e38
    v = torch.full((1, 2000, 1, 64), top, device=dev).to(dt)
    v[..., ::2] *= -1
    o = ops.block_attention(q, k, v, blocks).double()
    want = v[:, :1].double()
    # the denominator and the numerator add up the same terms: (2000 + 2) 2^-24 each at the most, 2^-17 for the terms, the last rounding
    assert ((o - want).abs() <= (torch.finfo(dt).eps + 2.0 ** -12) * want.abs()).all()


def test_forward_mode_derivatives_are_refused(dev):
    """The kernels have no forward-mode derivative: an input that carries a tangent is refused, not taken for a constant."""
    import torch.autograd.forward_ad as fw
    ops = pkg("network.operations")
    gen = torch.Generator(device=dev).manual_seed(1)
    q, k, v = _randn(gen, 1, 4, 2, 16), _randn(gen, 1, 130, 1, 16), _randn(gen, 1, 130, 1, 16)
    kq, w = _randn(gen, 1, 4, 1, 16), _randn(gen, 16)
    pos, freq = torch.arange(4.0, device=dev).view(1, 4), ops.rotation_frequencies(1, 8, device=dev)
    blocks = torch.zeros((1, 4, 1, 2), dtype=torch.int32, device=dev)
    calls = [(lambda *a: ops.norm_rotate(*a)[0], (q, kq, w, w, pos, freq)),
             (lambda *a: ops.block_attention(*a, blocks), (q, k, v)),
             (lambda *a: ops.sparse_attention(*a, 2), (q, k, v))]
    for call, args in calls:
        plain = call(*args)
        with fw.dual_level():
            assert torch.equal(call(*args), plain)                          # (no tangents: as ever)
            for i in range(len(args)):
                some = [fw.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match="tangent|forward"):
                    call(*some)
    # a tangent in the gradient that a backward pass starts from
    for call, args in calls[:2]:
        leaf = args[0].clone().requires_grad_()
        out = call(leaf, *args[1:])
        with fw.dual_level():
            go = fw.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="tangent|forward"):
                torch.autograd.grad(out, leaf, go)


def test_kept_means_behind_the_newest_rows_are_left(dev):
    """block_means(out=, last=) forms the blocks that hold the newest rows; those before and behind them keep what they hold."""
    ops = pkg("network.operations")
    gen = torch.Generator(device=dev).manual_seed(3)
    k = _randn(gen, 5, 400, 2, 32)
    live = [64, 100, 65, 400, 0]
    lens = torch.tensor(live, dtype=torch.int32, device=dev)
    for last in (1, 2, 64, 65, 130, 1000):
        out = torch.full((5, 7, 2, 32), 7.0, device=dev)
        ops.block_means(k, lens, out=out, last=last)
        want = orc64.means(k, lens).float()
        for e, n in enumerate(live):
            first, end = max(0, n - last) // 64, -(-n // 64)
            assert torch.equal(out[e, first:end], want[e, first:end])
            assert (out[e, :first] == 7).all() and (out[e, end:] == 7).all()


def test_from_two_threads(dev):
    """Calls of the same kernels with small and large workgroup memory from two threads, each on its own stream."""
    ops = pkg("network.operations")
    few = _inputs(dev, 1, 64, 4096, 1, 1, 64, 1, torch.bfloat16, 70)
    many = _inputs(dev, 1, 64, 4096, 1, 1, 64, 64, torch.bfloat16, 71)
    want = [_run(ops, s[:3], s[3], s[4]) for s in (few, many)]
    torch.cuda.synchronize()
    wrong = []

    def work(i, s):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(300):
                    got = _run(ops, s[:3], s[3], s[4])
                torch.cuda.current_stream().synchronize()
                wrong.extend(i for a, c in zip(got, want[i]) if not torch.equal(a, c))
        except RuntimeError as e:
            wrong.append(e)
    threads = [threading.Thread(target=work, args=x) for x in enumerate((few, many))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m,n,hq,hk,d,causal", [(200, 300, 4, 2, 64, False), (150, 150, 2, 2, 128, True), (100, 500, 3, 1, 24, False)])
def test_large_scores_that_are_rounded(dev, dtype, m, n, hq, hk, d, causal):
    """Random scores of 2^29 (fp16) to 2^62: the passes over queries and over keys form the same rounded scores, so that the largest
    key's probability is 1 in all of them: the output is its value, dv the sum of the gradients of the rows that chose it."""
    ops = pkg("network.operations")
    gen = torch.Generator(device=dev).manual_seed(7)
    dt = TYPES[dtype]
    big = 2.0 ** (12 if dt == torch.float16 else 30)
    q, k = (big * _randn(gen, 1, m, hq, d)).to(dt), (big * _randn(gen, 1, n, hk, d)).to(dt)
    v = torch.randint(-8, 9, (1, n, hk, d), device=dev, generator=gen).to(dt)
    go = torch.randint(-1, 2, (1, m, hq, d), device=dev, generator=gen).to(dt)
    blocks = torch.arange(-(-n // 64), dtype=torch.int32, device=dev).expand(1, m, hk, -1)
    o, _, _, dv = _run(ops, (q, k, v), go, blocks, 1.0, causal=causal)
    x = q.double().transpose(1, 2) @ k.double().transpose(1, 2).transpose(2, 3).contiguous().repeat_interleave(hq // hk, dim=1)
    if causal:
        x = torch.where(torch.arange(n, device=dev) <= torch.arange(m, device=dev)[:, None], x, torch.full_like(x, -math.inf))
    two, best = x.topk(2, dim=3) if not causal else x[:, :, 1:].topk(2, dim=3)
    # d + 8 roundings of at most d big^2 16 in both scores: the nearest two keys of a row are further apart than that
    assert ((two[..., 0] - two[..., 1]) > 2 * (d + 8) * 2.0 ** -24 * d * 16 * big * big).float().mean() > 0.99
    sure = (two[..., 0] - two[..., 1]) > 2 * (d + 8) * 2.0 ** -24 * d * 16 * big * big                          # (1,Hq,M)
    if causal:
        best = torch.cat((torch.zeros_like(best[:, :, :1]), best), dim=2)
        sure = torch.cat((torch.ones_like(sure[:, :, :1]), sure), dim=2)
    best = best[..., 0]
    for h in range(hq):
        want = v[0, best[0, h], h // (hq // hk)]
        assert torch.equal(o[0, sure[0, h], h], want[sure[0, h]])
    if bool(sure.all()):
        want = torch.zeros((1, n, hk, d), device=dev, dtype=torch.float64)
        for h in range(hq):
            want[0, :, h // (hq // hk)].index_add_(0, best[0, h], go[0, :, h].double())
        assert torch.equal(dv.double(), want)
    assert torch.isfinite(dv).all()


@pytest.mark.parametrize("b,m,n,hq,hk,d,count,causal", [(3, 400, 700, 2, 2, 24, 3, False), (2, 300, 1024, 4, 2, 64, 6, False),
                                                        (1, 600, 600, 6, 2, 128, 4, True)])
def test_errors_of_fp32(dev, b, m, n, hq, hk, d, count, causal):
    """Both forms round every score, difference, exponential, product and sum in fp32, the kernels a probability twice (its power, its
    quotient): the errors are of one size.  (With the log2 of the sum inside the exponent, half a step of 8 is a probability's whole
    error and more: gradients off by 1.9 times the plain form's.)"""
    ops = pkg("network.operations")
    q, k, v, go, blocks = _inputs(dev, b, m, n, hq, hk, d, count, torch.float32, 11)
    if causal:
        blocks[..., 0] = 0
    want = _formula(q, k, v, blocks, d ** -0.5, causal, go, torch.float64)
    plain = _formula(q, k, v, blocks, d ** -0.5, causal, go, torch.float32)
    for name, x, y, z in zip(("o", "dq", "dk", "dv"), _run(ops, (q, k, v), go, blocks, causal=causal), plain, want):
        here, there = _error(x, z), _error(y, z)
        print("%s: %.3g, plain %.3g" % (name, here, there))
        assert here <= 1.5 * there, (name, here, there)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["places", "coordinates"])
def test_errors_of_fp32_rotations(dev, kind, interleaved):
    """Against the plain form: angles, cosines and sines in 64 bits, everything else in fp32.  The kernel rounds its cosines and sines
    as the plain form does (a turn's last bits behind fp32 go in to first order), its products once less: the errors are of one
    size.  (With the turn alone in fp32 the angle was off by up to 2 pi 2^-26: outputs by 1.2 times the plain form's.)"""
    ops = pkg("network.operations")
    gen = torch.Generator(device=dev).manual_seed(9)
    b, n, h, d = 2, 900, 4, 64
    x, g, w = _randn(gen, b, n, h, d).requires_grad_(), _randn(gen, b, n, h, d), 1 + 0.2 * _randn(gen, d)
    if kind == "places":
        pos, freq = torch.randint(0, 100000, (b, n), device=dev, generator=gen), ops.rotation_frequencies(1, 32, device=dev)
    else:
        pos, freq = _randn(gen, b, n, 3), 2.0 ** torch.arange(10, device=dev, dtype=torch.float64).mul(0.6).repeat(3, 1)
    y, _ = ops.norm_rotate(x, None, w, None, pos, freq, interleaved=interleaved)
    dx, = torch.autograd.grad(y, x, g)
    ref = orc64.norm_rotate(x, w, pos, freq, 1e-6, interleaved, g)
    p = pos.double() if pos.dim() == 3 else pos.double().unsqueeze(2)
    a = (p.unsqueeze(3) * freq).flatten(2).unsqueeze(2)
    c, s, r = torch.cos(a).float(), torch.sin(a).float(), a.size(3)

    def turn(t, s):
        one, two = (t[..., 0:2 * r:2], t[..., 1:2 * r:2]) if interleaved else (t[..., :r], t[..., r:2 * r])
        pair = one * c - two * s, one * s + two * c
        return torch.cat((torch.stack(pair, dim=4).flatten(3) if interleaved else torch.cat(pair, dim=3), t[..., 2 * r:]), dim=3)
    xf = x.detach()
    inv = torch.rsqrt((xf * xf).mean(dim=3, keepdim=True) + 1e-6)
    unit, back = xf * inv, turn(g, -s) * w
    for name, got, plain, want in (("y", y, turn(unit * w, s), ref["y"]),
                                   ("dx", dx, inv * (back - unit * (back * unit).mean(dim=3, keepdim=True)), ref["dx"])):
        here, there = _error(got, want), _error(plain, want)
        print("%s: %.3g, plain %.3g" % (name, here, there))
        assert here <= 1.1 * there, (name, here, there)
