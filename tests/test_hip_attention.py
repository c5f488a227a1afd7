"""gpu: norm_rotate, block_means, select_blocks, block_attention and sparse_attention against their definitions in 64 bits
(attention_oracle.py, which also derives the bounds), at the sizes and masks where such kernels go wrong."""
import math

import pytest
import torch

import attention_oracle as orc64
from conftest import pkg

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, device=gen.device, generator=gen).to(dtype)


def _within(got, want, bound, what):
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() / bound.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert over <= 1.0, "%s: %.3g of its bound" % (what, over)


# ---- norm_rotate -------------------------------------------------------------------------------------------------------
NORM = [  # b, n, hq, hk, d, axes, pairs, weights, interleaved, position
    (1, 1, 1, 1, 8, 1, 4, "one", False, "i32"),
    (3, 1, 16, 4, 128, 1, 64, "one", False, "i64"),
    (2, 17, 3, 1, 24, 3, 3, "head", False, "f32"),
    (2, 33, 4, 2, 32, 3, 5, "head", True, "f32"),
    (1, 313, 5, 2, 40, 2, 7, "one", False, "f64"),
    (2, 70, 2, 2, 64, 1, 32, "none", True, "i32"),
    (1, 65, 3, 3, 80, 1, 11, "mixed", False, "i32"),
    (1, 129, 6, 1, 96, 2, 24, "head", False, "f32"),
    (1, 40, 2, 1, 256, 1, 128, "head", False, "i32"),
    (1, 40, 2, 1, 200, 3, 33, "one", True, "f32"),
    (2, 2000, 7, 1, 64, 3, 10, "head", False, "f32"),
    (4, 1500, 2, 2, 64, 3, 10, "one", False, "f32"),
    (1, 70, 127, 2, 128, 1, 64, "head", False, "i32"),
]


def _norm_inputs(dev, case, dtype, seed=5):
    b, n, hq, hk, d, axes, pairs, weights, interleaved, pos = case
    gen = _gen(dev, seed)
    q, k = _randn(gen, b, n, hq, d, dtype=dtype), _randn(gen, b, n, hk, d, dtype=dtype)
    q[0, 0, 0] = 0                                                          # a row of zeros: eps alone
    wt = dtype if weights == "mixed" else torch.float32
    shape = {"one": ((d,), (d,)), "head": ((hq, d), (hk, d)), "mixed": ((d,), (hk, d)), "none": (None, None)}[weights]
    w = [None if s is None else (1 + 0.3 * _randn(gen, *s)).to(wt) for s in shape]
    if pos in ("i32", "i64"):
        position = torch.randint(0, 1 << 20, (b, n, axes), device=dev, generator=gen).to(torch.int32 if pos == "i32" else torch.int64)
        position = position[:, :, 0] if axes == 1 else position
    else:
        position = 3 * _randn(gen, b, n, axes, dtype=torch.float64 if pos == "f64" else torch.float32)
    freq = pkg("network.operations").rotation_frequencies(axes, pairs, device=dev)
    return q, k, w[0], w[1], position, freq, interleaved


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("case", range(len(NORM)))
def test_norm_rotate_forward_and_gradients(dev, case, dtype):
    ops = pkg("network.operations")
    q, k, wq, wk, position, freq, inter = _norm_inputs(dev, NORM[case], TYPES[dtype])
    leaves = [t for t in (q, k, wq, wk) if t is not None]
    for t in leaves:
        t.requires_grad_()
    oq, ok = ops.norm_rotate(q, k, wq, wk, position, freq, interleaved=inter)
    gen = _gen(dev, 6)
    gq, gk = _randn(gen, *q.shape, dtype=q.dtype), _randn(gen, *k.shape, dtype=k.dtype)
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad((oq, ok), leaves, (gq, gk))))
    for x, w, o, g, nm in ((q, wq, oq, gq, "q"), (k, wk, ok, gk, "k")):
        ref = orc64.norm_rotate(x, w, position, freq, 1e-6, inter, g)
        assert o.dtype == x.dtype and grads[id(x)].dtype == x.dtype
        _within(o, ref["y"], ref["t_y"], nm)
        _within(grads[id(x)], ref["dx"], ref["t_dx"], "d" + nm)
        if w is not None:
            assert grads[id(w)].dtype == w.dtype
            _within(grads[id(w)], ref["dw"], ref["t_dw"], "weight of " + nm)


def test_norm_rotate_strided_broadcast_and_single_side(dev):
    """Slices of a fused projection, a broadcast input, rows off the 16-byte grid, no keys, weights without a gradient."""
    ops = pkg("network.operations")
    gen = _gen(dev, 9)
    fused = _randn(gen, 2, 50, 8, 48, dtype=torch.bfloat16).requires_grad_()
    q, k = fused[:, :, :5], fused[:, :, 5:7]
    position, freq = torch.randint(0, 99, (2, 50), device=dev, generator=gen), ops.rotation_frequencies(1, 24, device=dev)
    oq, ok = ops.norm_rotate(q, k, None, None, position, freq)
    ref = [orc64.norm_rotate(t, None, position, freq, g=torch.ones_like(t)) for t in (q, k)]
    _within(oq, ref[0]["y"], ref[0]["t_y"], "q"), _within(ok, ref[1]["y"], ref[1]["t_y"], "k")
    grad, = torch.autograd.grad(oq.sum() + ok.sum(), fused)
    _within(grad[:, :, :5], ref[0]["dx"], ref[0]["t_dx"], "dq")
    _within(grad[:, :, 5:7], ref[1]["dx"], ref[1]["t_dx"], "dk")
    assert (grad[:, :, 7] == 0).all()
    one = _randn(gen, 2, 1, 3, 48)
    wide = one.expand(2, 50, 3, 48)
    odd = torch.empty(2 * 50 * 3 * 48 + 1, device=dev)[1:].view(2, 50, 3, 48).copy_(wide)
    w = 1 + 0.1 * _randn(gen, 48)
    a, none = ops.norm_rotate(wide, None, w, None, position, freq, interleaved=True)
    c, _ = ops.norm_rotate(odd, None, w, None, position, freq, interleaved=True)
    assert none is None and torch.equal(a, c)
    ref = orc64.norm_rotate(wide, w, position, freq, 1e-6, True)
    _within(a, ref["y"], ref["t_y"], "broadcast")
    # one pair fewer than the channels: what is behind the pairs passes; no pairs at all: the norm alone
    b0, _ = ops.norm_rotate(odd, None, w, None, position, freq[:, :0])
    _within(b0, orc64.norm_rotate(odd, w, position, freq[:, :0])["y"], ref["t_y"] + 1e-6, "no pairs")
    for shape in ((0, 4, 2, 16), (3, 0, 2, 16)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        ww = torch.ones(16, device=dev, requires_grad=True)
        y, _ = ops.norm_rotate(x, None, ww, None, torch.zeros(shape[:2], device=dev), ops.rotation_frequencies(1, 8, device=dev))
        gx, gw = torch.autograd.grad(y.sum(), (x, ww))
        assert y.shape == shape and gx.shape == shape and (gw == 0).all()


def test_norm_rotate_gradient_against_differences(dev):
    """sum(g * f(x + t e)) - sum(g * f(x - t e)) over 2 t in fp32: the third derivative and the fp32 noise (2^-24 of the sum
    of |g f|, over t) are both below 1e-3 of |grad| |e| at t = 1e-2."""
    ops = pkg("network.operations")
    q, k, wq, wk, position, freq, inter = _norm_inputs(dev, (2, 40, 3, 2, 48, 3, 8, "head", False, "f32"), torch.float32)
    q[0, 0, 0] = 1.0
    gen = _gen(dev, 3)
    gq, gk = _randn(gen, *q.shape), _randn(gen, *k.shape)
    leaves = [q, k, wq, wk]
    steps = [_randn(gen, *t.shape) for t in leaves]

    def loss(sign):
        ts = [t + sign * 1e-2 * s for t, s in zip(leaves, steps)]
        oq, ok = ops.norm_rotate(*ts, position, freq, interleaved=inter)
        return ((oq.double() * gq).sum() + (ok.double() * gk).sum()).item()
    got = (loss(1) - loss(-1)) / 2e-2
    for t in leaves:
        t.requires_grad_()
    grads = torch.autograd.grad(ops.norm_rotate(*leaves, position, freq, interleaved=inter), leaves, (gq, gk))
    want = sum((g.double() * s).sum().item() for g, s in zip(grads, steps))
    size = math.sqrt(sum((g.double() ** 2).sum().item() for g in grads)) * math.sqrt(sum((s.double() ** 2).sum().item() for s in steps))
    assert abs(got - want) < 1e-3 * size


# ---- blocks ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("b,n,hk,d,ragged", [(2, 1, 1, 8, False), (3, 63, 2, 24, False), (2, 64, 3, 128, True), (4, 200, 1, 64, True),
                                             (1, 1000, 8, 96, False), (2, 130, 40, 128, True)])
def test_block_means(dev, b, n, hk, d, ragged, dtype):
    ops = pkg("network.operations")
    gen = _gen(dev, 1)
    k = _randn(gen, b, n, hk, d, dtype=TYPES[dtype])
    n_arr = None
    if ragged:
        n_arr = torch.tensor([0, n, 1, n // 2][:b], dtype=torch.int32, device=dev)
        for e in range(b):
            k[e, int(n_arr[e]):] = math.nan                                 # behind the live rows: never read
    got = ops.block_means(k, n_arr)
    want = orc64.means(k, n_arr)
    assert got.dtype == torch.float32 and torch.equal(got, want.float())


def test_block_means_of_a_growing_cache(dev):
    ops = pkg("network.operations")
    gen = _gen(dev, 2)
    k = _randn(gen, 3, 700, 2, 32, dtype=torch.float16)
    old = torch.tensor([100, 630, 64], dtype=torch.int32, device=dev)
    out = ops.block_means(k, old)
    for step in (1, 70):
        new = old + step
        kept = out.clone()
        ops.block_means(k, new, out=out, last=step)
        want = ops.block_means(k, new)
        assert torch.equal(out, want)
        for e in range(3):
            first = int(old[e]) // 64
            assert torch.equal(out[e, :first], kept[e, :first])
        old = new
    poison = torch.full_like(out, 7.0)
    ops.block_means(k, old, out=poison, last=0)
    assert (poison == 7.0).all()


SELECT = [  # b, m, n, hq, hk, d, count, causal, ragged
    (1, 1, 1, 1, 1, 8, 1, False, False),
    (1, 1, 1, 1, 1, 8, 3, True, False),
    (2, 70, 130, 4, 2, 24, 2, False, False),
    (2, 130, 130, 6, 2, 64, 1, True, False),
    (2, 130, 130, 2, 2, 64, 2, True, True),
    (3, 50, 640, 3, 1, 40, 5, False, True),
    (1, 300, 1500, 8, 8, 128, 16, True, False),
    (2, 1, 66000, 8, 2, 128, 16, True, True),
    (1, 2, 90000, 2, 1, 32, 64, False, False),
    (1, 1, 140000, 1, 1, 16, 7, False, False),
    (1, 200, 4200, 2, 2, 64, 64, False, True),
    (1, 700, 5000, 4, 2, 64, 8, False, False),
    (2, 2100, 5000, 2, 1, 24, 13, True, True),
    (9, 500, 300, 1, 1, 8, 3, False, False),
    (1, 2100, 1500, 8, 2, 128, 16, True, False),
    (1, 2200, 4200, 2, 2, 64, 64, False, True),
    (3, 710, 2000, 6, 2, 40, 30, True, True),
    (2, 1100, 9000, 4, 4, 96, 6, False, True),
    (1, 4200, 4200, 1, 1, 16, 1, True, False),
    (1, 8300, 66000, 1, 1, 32, 5, False, False),
]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("case", range(len(SELECT)))
def test_select_blocks(dev, case, dtype):
    ops = pkg("network.operations")
    b, m, n, hq, hk, d, count, causal, ragged = SELECT[case]
    gen = _gen(dev, 4 + case)
    q = _randn(gen, b, m, hq, d, dtype=TYPES[dtype])
    mean = 0.1 * _randn(gen, b, -(-n // 64), hk, d)
    n_arr = m_arr = None
    if ragged:
        n_arr = torch.tensor([n, n // 3, 0][:b], dtype=torch.int32, device=dev)
        m_arr = torch.tensor([m, min(m, n // 3), 0][:b][::-1] if not causal else [m, min(m, n // 3), 0][:b], dtype=torch.int32, device=dev)
        for e in range(b):
            q[e, int(m_arr[e]):] = math.nan
            mean[e, -(-int(n_arr[e]) // 64):] = math.nan
    got = ops.select_blocks(q, mean, n, count, n_arr, m_arr, causal)
    want = orc64.select(q, mean, n, count, n_arr, m_arr, causal)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("m", [1, 3, 400, 2200])
def test_select_blocks_ties_and_not_numbers(dev, m):
    """Equal means, equal scores of opposite signs, zero queries: the lowest block wins; NaN ranks behind every number and
    infinities rank as such; means whose scores differ by less than an fp32 rounding keep their order."""
    ops = pkg("network.operations")
    gen = _gen(dev, 8)
    n, d, count = 64 * 100, 32, 9
    q = _randn(gen, 2, m, 1, d)
    q[0, 0] = 0
    mean = _randn(gen, 2, 100, 1, d)
    mean[:, 40:80] = mean[:, 0:40]                                          # every block twice
    mean[1, 3] = math.nan
    mean[1, 90, 0, 0] = math.inf
    mean[1, 91, 0, 0] = -math.inf
    near = mean[0, 10].clone()
    mean[0, 95] = near
    mean[0, 95, 0, 5] = torch.nextafter(near[0, 5], near[0, 5] + 1)         # one fp32 step away
    got = ops.select_blocks(q, mean, n, count)
    assert torch.equal(got.cpu(), orc64.select(q, mean, n, count))
    assert got[0, 0, 0].tolist() == list(range(count))
    flat = torch.zeros_like(mean)
    assert (ops.select_blocks(q, flat, n, count)[..., :] == torch.arange(count, device=dev)).all()
    nan = torch.full_like(mean, math.nan)
    assert torch.equal(ops.select_blocks(q, nan, n, 100 % 65)[..., :3], torch.arange(3, device=dev, dtype=torch.int32).expand(2, m, 1, 3))


@pytest.mark.parametrize("kind", ["tiny queries", "tiny means", "heads that cancel", "far apart"])
def test_select_blocks_at_the_ends_of_the_range(dev, kind):
    """Squares that leave fp32's range, and heads whose sum is far smaller than they are: what the approximate scores are off
    by must not be taken for less than it is."""
    ops = pkg("network.operations")
    gen = _gen(dev, 18)
    q, mean = _randn(gen, 1, 4200, 2, 40), _randn(gen, 1, 90, 1, 40)
    if kind == "tiny queries":
        q *= 1e-24
    elif kind == "tiny means":
        mean *= 1e-27
    elif kind == "heads that cancel":
        q[:, :, 1] = 1e-3 * q[:, :, 1] - 1e4 * q[:, :, 0]
        q[:, :, 0] *= 1e4
    else:
        q[:, ::2] *= 1e15
        mean[:, 1::3] *= 1e-18
    got = ops.select_blocks(q, mean, 90 * 64, 6)
    assert torch.equal(got.cpu(), orc64.select(q, mean, 90 * 64, 6))


@pytest.mark.parametrize("m", [7, 4300])
def test_select_blocks_zeros_and_queries_that_are_not_numbers(dev, m):
    """Queries and means with one channel each: most scores are exactly 0, of either sign.  Rows of NaN and infinities: the
    scores that are numbers first."""
    ops = pkg("network.operations")
    gen = _gen(dev, 28)
    q, mean = torch.zeros((1, m, 1, 24), device=dev), torch.zeros((1, 70, 1, 24), device=dev)
    q[0, torch.arange(m), 0, torch.randint(0, 24, (m,), device=dev, generator=gen)] = 1.0
    mean[0, torch.arange(70), 0, torch.randint(0, 24, (70,), device=dev, generator=gen)] = torch.randn(70, device=dev, generator=gen)
    mean[0, ::5] *= -1
    q[0, 3] = math.nan
    q[0, 5, 0, 1] = math.inf
    if m > 100:
        q[0, 70:90] = math.nan
        q[0, 200:210] = 0
    for count in (3, 20):
        got = ops.select_blocks(q, mean, 70 * 64, count)
        assert torch.equal(got.cpu(), orc64.select(q, mean, 70 * 64, count))


# ---- attention ---------------------------------------------------------------------------------------------------------
ATTEND = [  # b, m, n, hq, hk, d, count, causal, ragged
    (1, 1, 1, 1, 1, 8, 1, False, False),
    (2, 1, 65, 2, 1, 16, 2, True, False),
    (2, 63, 64, 2, 2, 24, 1, False, False),
    (2, 65, 130, 4, 2, 32, 2, False, True),
    (2, 130, 130, 3, 1, 40, 2, True, False),
    (3, 100, 200, 6, 2, 64, 3, True, True),
    (1, 129, 640, 5, 1, 80, 4, False, False),
    (1, 312, 312, 4, 4, 96, 5, False, False),
    (1, 200, 400, 8, 2, 128, 4, True, False),
    (2, 5, 1000, 64, 1, 64, 7, False, True),
    (1, 9, 300, 7, 1, 128, 3, True, False),
    (1, 70, 4300, 2, 2, 32, 64, False, False),
    (2, 1, 3000, 8, 2, 128, 16, True, True),
    (1, 1000, 300, 2, 2, 64, 2, False, False),
    (1, 4500, 130, 1, 1, 8, 2, False, False),
    (1, 4300, 200, 2, 1, 64, 3, True, False),
    (2, 70, 4160, 8, 8, 32, 5, False, True),
]


def _attend_inputs(dev, case, dtype, seed=20):
    b, m, n, hq, hk, d, count, causal, ragged = case
    gen = _gen(dev, seed)
    q, k, v = _randn(gen, b, m, hq, d, dtype=dtype), _randn(gen, b, n, hk, d, dtype=dtype), _randn(gen, b, n, hk, d, dtype=dtype)
    go = _randn(gen, b, m, hq, d, dtype=dtype)
    nb = -(-n // 64)
    # any order, names twice, names outside
    blocks = torch.randint(-1, nb + 2, (b, m, hk, count), device=dev, generator=gen).to(torch.int32)
    blocks[:, :, :, 0] = torch.randint(0, nb, (b, m, hk), device=dev, generator=gen).to(torch.int32)
    if m > 2:
        blocks[0, m // 2] = -1                                              # a query that names nothing
    n_arr = m_arr = None
    if ragged:
        n_arr = torch.tensor([n, n // 2, 0][:b], dtype=torch.int32, device=dev)
        m_arr = torch.tensor([m, max(1, m // 2), m][:b], dtype=torch.int32, device=dev)
        for e in range(b):
            for t in (k, v):
                t[e, int(n_arr[e]):] = math.nan
            for t in (q, go):
                t[e, int(m_arr[e]):] = math.inf
    return q, k, v, go, blocks, n_arr, m_arr


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_block_attention_forward_and_gradients(dev, case, dtype):
    ops = pkg("network.operations")
    causal = ATTEND[case][7]
    q, k, v, go, blocks, n_arr, m_arr = _attend_inputs(dev, ATTEND[case], TYPES[dtype])
    with torch.no_grad():
        plain = ops.block_attention(q, k, v, blocks, None, n_arr, m_arr, causal)
    for t in (q, k, v):
        t.requires_grad_()
    o = ops.block_attention(q, k, v, blocks, None, n_arr, m_arr, causal)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), go)
    ref = orc64.attention(q, k, v, blocks, None, n_arr, m_arr, causal, go)
    assert torch.equal(plain, o.detach()) and o.dtype == q.dtype
    for nm, t in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        _within(t, ref[nm], ref["t_" + nm], nm)
    see = orc64.seen(q.size(0), q.size(1), k.size(1), k.size(2), blocks, n_arr, m_arr, causal)
    nothing = ~see.any(dim=3).transpose(1, 2).repeat_interleave(q.size(2) // k.size(2), dim=2)
    assert (o[nothing] == 0).all() and (dq[nothing] == 0).all()
    assert (dk[~see.any(dim=2).transpose(1, 2)] == 0).all() and (dv[~see.any(dim=2).transpose(1, 2)] == 0).all()
    # the same bits every time: nothing is added up in the order of arrival
    again = torch.autograd.grad(ops.block_attention(q, k, v, blocks, None, n_arr, m_arr, causal), (q, k, v), go)
    assert all(torch.equal(a, c) for a, c in zip((dq, dk, dv), again))


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_block_attention_small_and_large_values(dev, dtype):
    """Gradients of 1e-4 beside those of 1 (fp16: their products with probabilities are below its normal numbers), scores of
    +-80, a scale of its own."""
    ops = pkg("network.operations")
    q, k, v, go, blocks, _, _ = _attend_inputs(dev, (1, 150, 512, 2, 1, 64, 6, False, False), TYPES[dtype], 31)
    go[:, ::2] *= 1e-4
    for scale in (0.9, 1e-3):
        for t in (q, k, v):
            t.requires_grad_()
        o = ops.block_attention(q, k, v, blocks, scale)
        grads = torch.autograd.grad(o, (q, k, v), go)
        ref = orc64.attention(q, k, v, blocks, scale, go=go)
        for nm, t in zip(("o", "dq", "dk", "dv"), (o,) + grads):
            _within(t, ref[nm], ref["t_" + nm], nm)


def test_block_attention_strides_types_and_empty(dev):
    ops = pkg("network.operations")
    gen = _gen(dev, 40)
    fused = _randn(gen, 2, 100, 8, 48, dtype=torch.bfloat16).requires_grad_()
    q, k, v = fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:]
    blocks = torch.tensor([0, 1], device=dev).expand(2, 100, 2, 2)          # int64, stride 0
    o = ops.block_attention(q, k, v, blocks, causal=True)
    dense = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    o2 = ops.block_attention(*dense, blocks.to(torch.int32).contiguous(), causal=True)
    assert torch.equal(o, o2)
    go = _randn(gen, *o.shape, dtype=o.dtype)
    grad, = torch.autograd.grad(o, fused, go)
    assert torch.equal(grad, torch.cat(torch.autograd.grad(o2, dense, go), dim=2))
    # heads first in memory, a broadcast gradient, keys shared by two sequences
    hf = [t.detach().transpose(1, 2).contiguous().transpose(1, 2) for t in dense]
    assert torch.equal(ops.block_attention(*hf, blocks, causal=True), o2)
    one = torch.autograd.grad(ops.block_attention(*dense, blocks, causal=True).sum(), dense)      # (gradient of stride 0)
    ref = orc64.attention(*dense, blocks, causal=True, go=torch.ones_like(o2))
    for nm, t in zip(("dq", "dk", "dv"), one):
        _within(t, ref[nm], ref["t_" + nm], nm)
    shared = dense[1].detach()[:1].expand(2, 100, 2, 48).requires_grad_()
    o3 = ops.block_attention(dense[0].detach(), shared, dense[2].detach(), blocks)
    ref = orc64.attention(dense[0], shared, dense[2], blocks)
    _within(o3, ref["o"], ref["t_o"], "shared keys")
    # blocks far outside 32 bits name nothing
    far = torch.full((2, 100, 2, 1), 1 << 32, device=dev)
    assert (ops.block_attention(*[t.detach() for t in dense], far) == 0).all()
    for b, m, n in ((0, 3, 70), (2, 0, 70), (2, 3, 0)):
        ts = [torch.ones((b, m, 2, 16), device=dev), torch.ones((b, n, 1, 16), device=dev), torch.ones((b, n, 1, 16), device=dev)]
        for t in ts:
            t.requires_grad_()
        o = ops.block_attention(*ts, torch.zeros((b, m, 1, 1), dtype=torch.int32, device=dev))
        grads = torch.autograd.grad(o.sum(), ts)
        assert (o == 0).all() and o.shape == ts[0].shape and all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, ts))
        s = ops.sparse_attention(*[t.detach() for t in ts], 2)
        assert (s == 0).all() and s.shape == o.shape


def test_block_attention_gradient_against_differences(dev):
    """As for norm_rotate: central differences of an fp32 forward, t = 1e-2, within 1e-3 of |grad| |step|."""
    ops = pkg("network.operations")
    q, k, v, go, blocks, _, _ = _attend_inputs(dev, (1, 60, 200, 4, 2, 32, 3, True, False), torch.float32, 51)
    gen = _gen(dev, 52)
    leaves = [q, k, v]
    steps = [_randn(gen, *t.shape) for t in leaves]

    def loss(sign):
        ts = [t + sign * 1e-2 * s for t, s in zip(leaves, steps)]
        return (ops.block_attention(*ts, blocks, causal=True).double() * go).sum().item()
    got = (loss(1) - loss(-1)) / 2e-2
    for t in leaves:
        t.requires_grad_()
    grads = torch.autograd.grad(ops.block_attention(*leaves, blocks, causal=True), leaves, go)
    want = sum((g.double() * s).sum().item() for g, s in zip(grads, steps))
    size = math.sqrt(sum((g.double() ** 2).sum().item() for g in grads)) * math.sqrt(sum((s.double() ** 2).sum().item() for s in steps))
    assert abs(got - want) < 1e-3 * size


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_not_numbers_stay_where_they_are_seen(dev, dtype):
    """A key or value that is not finite reaches the queries that see it and no other: not those that picked other blocks,
    not the earlier ones of its own block under a causal mask; forward and dq."""
    ops = pkg("network.operations")
    q, k, v, go, _, _, _ = _attend_inputs(dev, (1, 128, 192, 2, 1, 64, 2, True, False), TYPES[dtype], 61)
    blocks = torch.zeros((1, 128, 1, 2), dtype=torch.int32, device=dev)
    blocks[:, ::2, :, 1] = 1
    blocks[:, 1::2, :, 1] = 2
    for bad_k, bad_v in ((None, 70), (None, 150), (100, None), (180, 70)):
        kk, vv = k.clone(), v.clone()
        if bad_k is not None:
            kk[0, bad_k, 0, 3] = math.inf
        if bad_v is not None:
            vv[0, bad_v, 0, 5:9] = torch.tensor([math.nan, math.inf, -math.inf, math.nan], device=dev).to(v.dtype)
        leaves = [t.clone().requires_grad_() for t in (q, kk, vv)]
        o = ops.block_attention(*leaves, blocks, causal=True)
        dq, _, _ = torch.autograd.grad(o, leaves, go)
        see = orc64.seen(1, 128, 192, 1, blocks, causal=True)[0, 0]
        hit = torch.zeros(128, dtype=torch.bool, device=dev)
        for j in (bad_k, bad_v):
            if j is not None:
                hit |= see[:, j]
        assert hit.any() and not hit.all()
        clean = [t.clone().requires_grad_() for t in (q, k, v)]
        o2 = ops.block_attention(*clean, blocks, causal=True)
        dq2, _, _ = torch.autograd.grad(o2, clean, go)
        assert torch.equal(o[0, ~hit], o2[0, ~hit]) and torch.equal(dq[0, ~hit], dq2[0, ~hit])
        if bad_v is not None:
            sees_v = see[:, bad_v]
            assert not torch.isfinite(o[0, sees_v][..., 5:9]).any()
            assert not torch.isfinite(dq[0, sees_v]).all(dim=-1).any()
        if bad_k is not None:
            assert not torch.isfinite(dq[0, see[:, bad_k]]).all(dim=-1).any()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_not_numbers_of_queries_reach_the_keys_they_see(dev, dtype):
    """dk and dv: a query or an output gradient that is not finite reaches the keys that its query sees, not the later ones of
    the same block under a causal mask."""
    ops = pkg("network.operations")
    q, k, v, go, _, _, _ = _attend_inputs(dev, (1, 128, 192, 2, 1, 64, 2, True, False), TYPES[dtype], 62)
    blocks = torch.zeros((1, 128, 1, 2), dtype=torch.int32, device=dev)
    blocks[:, ::2, :, 1] = 1
    blocks[:, 1::2, :, 1] = 2
    see = orc64.seen(1, 128, 192, 1, blocks, causal=True)[0, 0]
    for which in (0, 1):
        for i in (20, 101):
            pair = [q.clone(), go.clone()]
            pair[which][0, i, 1, 7] = math.nan
            bad = [t.clone().requires_grad_() for t in (pair[0], k, v)]
            _, dk, dv = torch.autograd.grad(ops.block_attention(*bad, blocks, causal=True), bad, pair[1])
            pair[which][0, i, 1, 7] = 0
            clean = [t.clone().requires_grad_() for t in (pair[0], k, v)]
            _, dk2, dv2 = torch.autograd.grad(ops.block_attention(*clean, blocks, causal=True), clean, pair[1])
            hit = see[i]
            assert hit.any() and not hit.all() and not hit[(hit.nonzero().max() // 64 * 64):].all()
            assert torch.equal(dk[0, ~hit], dk2[0, ~hit]) and torch.equal(dv[0, ~hit], dv2[0, ~hit])
            assert dk[0, hit].isnan().any(dim=-1).all() and dv[0, hit].isnan().any(dim=-1).all()


def test_score_gradients_beyond_half_precision(dev):
    """fp16: do . v passes 65504 many times over although every input and every result is far below it."""
    ops = pkg("network.operations")
    q, k, v, go, blocks, _, _ = _attend_inputs(dev, (1, 150, 512, 2, 1, 128, 6, False, False), torch.float16, 33)
    gen = _gen(dev, 34)
    v = (8000 * torch.sign(_randn(gen, 1, 512, 1, 1)) + 100 * _randn(gen, 1, 512, 1, 128)).half()
    go = (1e-3 * (1 + 0.1 * _randn(gen, *go.shape))).half()
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = ops.block_attention(*leaves, blocks, 0.01)
    ref = orc64.attention(q, k, v, blocks, 0.01, go=go)
    for nm, t in zip(("o", "dq", "dk", "dv"), (o,) + torch.autograd.grad(o, leaves, go)):
        _within(t, ref[nm], ref["t_" + nm], nm)


def test_keys_behind_2_to_the_31_elements(dev):
    """One query over 2.2e9 elements of keys: the offsets pass 32 bits; blocks beyond 32768."""
    ops = pkg("network.operations")
    gen = _gen(dev, 70)
    n, hk, d, count = 2_150_000, 8, 128, 6
    k = torch.zeros((1, n, hk, d), dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    tail = 64 * 40 + 17
    k[:, n - tail:] = _randn(gen, 1, tail, hk, d, dtype=k.dtype)
    v[:, n - tail:] = _randn(gen, 1, tail, hk, d, dtype=k.dtype)
    q = _randn(gen, 1, 2, 16, d, dtype=k.dtype)
    means = ops.block_means(k)
    first = (n - tail) // 64
    assert (means[:, :first] == 0).all()
    assert torch.equal(means[:, first:], orc64.means(k[:, first * 64:]).float())
    blocks = ops.select_blocks(q, means, n, count, causal=True)
    want = orc64.select(q, means[:, first - 2:], n - (first - 2) * 64, count, causal=True)
    assert torch.equal(blocks.cpu(), want + first - 2)
    o = ops.block_attention(q, k, v, blocks, causal=True)
    ref = orc64.attention(q, k[:, first * 64:], v[:, first * 64:], blocks - first, causal=True)
    _within(o, ref["o"], ref["t_o"], "o")


# ---- together ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_between_points_as_one_layer(dev, dtype):
    """Points in a spatial order, queries and keys normed and turned by the coordinates, sparse attention, gradients down to
    the projections' outputs and the norms' weights; the oracle takes the operators' own intermediate tensors, so that the
    picked blocks are those of the same rounded queries."""
    ops = pkg("network.operations")
    gen = _gen(dev, 80)
    dt = TYPES[dtype]
    b, n, hq, hk, d, count = 2, 700, 4, 2, 32, 4
    xyz = torch.randn((b, n, 3), device=dev, generator=gen)
    xyz = torch.stack([c[c[:, 0].argsort()] for c in xyz])
    fused = _randn(gen, b, n, hq + 2 * hk, d, dtype=dt).requires_grad_()
    w = (1 + 0.1 * _randn(gen, 2, d)).requires_grad_()
    freq = 2.0 ** torch.arange(5, device=dev, dtype=torch.float64).repeat(3, 1)
    q0, k0, v = fused[:, :, :hq], fused[:, :, hq:hq + hk], fused[:, :, hq + hk:]
    q, k = ops.norm_rotate(q0, k0, w[0], w[1], xyz, freq)
    n_arr = torch.tensor([n, 401], dtype=torch.int32, device=dev)
    o = ops.sparse_attention(q, k, v, count, n_arr=n_arr, m_arr=n_arr)
    go = _randn(gen, *o.shape, dtype=dt)
    gf, gw = torch.autograd.grad(o, (fused, w), go)
    means = ops.block_means(k, n_arr)
    assert torch.equal(means, orc64.means(k, n_arr).float())
    blocks = ops.select_blocks(q, means, n, count, n_arr, n_arr)
    assert torch.equal(blocks.cpu(), orc64.select(q, means, n, count, n_arr, n_arr))
    ref = orc64.attention(q, k, v, blocks, None, n_arr, n_arr, go=go)
    _within(o, ref["o"], ref["t_o"], "o")
    _within(gf[:, :, hq + hk:], ref["dv"], ref["t_dv"], "dv")
    # the norms' gradient is linear in its input: the bound of dq and dk goes through it
    for x, ww, sl, nm, i in ((q0, w[0], slice(0, hq), "dq", 0), (k0, w[1], slice(hq, hq + hk), "dk", 1)):
        r = orc64.norm_rotate(x, ww, xyz, freq, g=ref[nm])
        slack = orc64.norm_rotate(x, ww, xyz, freq, g=ref["t_" + nm] + orc64.unit(dt) * ref[nm].abs())
        inv = 1 / torch.sqrt((x.detach().double() ** 2).mean(dim=3, keepdim=True) + 1e-6)
        reach = (ref["t_" + nm] + orc64.unit(dt) * ref[nm].abs()).norm(dim=3, keepdim=True) * ww.detach().double().abs().max() * inv * 2
        _within(gf[:, :, sl], r["dx"], r["t_dx"] + slack["t_dx"] + reach, nm)
        u = x.detach().double() * inv
        per_row = (ref["t_" + nm] + orc64.unit(dt) * ref[nm].abs()).norm(dim=3, keepdim=True)
        _within(gw[i], r["dw"], r["t_dw"] + (per_row * u.abs()).sum(dim=(0, 1, 2)), "weights of " + nm)


def test_single_tokens_over_a_kept_cache(dev):
    """A step of serving: a row is appended, its means are brought up to date, one query per sequence attends; every step
    equals the same row of a call over the whole sequence."""
    ops = pkg("network.operations")
    gen = _gen(dev, 90)
    b, n, hq, hk, d, count = 3, 260, 4, 2, 64, 3
    q, k, v = (_randn(gen, b, n, h, d, dtype=torch.float32) for h in (hq, hk, hk))
    whole = ops.sparse_attention(q, k, v, count, causal=True)
    kc, vc = torch.full_like(k, math.nan), torch.full_like(v, math.nan)
    kc[:, :190], vc[:, :190] = k[:, :190], v[:, :190]
    lens = torch.full((b,), 190, dtype=torch.int32, device=dev)
    means = ops.block_means(kc, lens)
    for t in range(190, n):
        kc[:, t], vc[:, t] = k[:, t], v[:, t]
        lens += 1
        ops.block_means(kc, lens, out=means, last=1)
        o = ops.sparse_attention(q[:, t:t + 1], kc, vc, count, n_arr=lens, causal=True, means=means)
        # (the means of the query's own block are not scored, so the picked blocks are the same)
        ref = orc64.attention(q[:, t:t + 1], k[:, :t + 1], v[:, :t + 1],
                              ops.select_blocks(q[:, t:t + 1], means[:, :t // 64 + 1], t + 1, count, causal=True), causal=True)
        _within(o, ref["o"], ref["t_o"], "o")
        assert (o - whole[:, t:t + 1]).abs().max() <= 2 * ref["t_o"].max()


# ---- streams, graphs, devices ------------------------------------------------------------------------------------------
def test_on_side_streams_at_once(dev):
    ops = pkg("network.operations")
    sets = [_attend_inputs(dev, (2, 150, 600, 4, 2, 64, 4, False, False), torch.bfloat16, 100 + i) for i in range(2)]
    want = []
    for q, k, v, go, blocks, _, _ in sets:
        for t in (q, k, v):
            t.requires_grad_()
        o = ops.block_attention(q, k, v, blocks)
        want.append((o.detach(),) + torch.autograd.grad(o, (q, k, v), go))
    few = [ops.sparse_attention(s[0][:, :1].detach(), s[1].detach(), s[2].detach(), 3) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                q, k, v, go, blocks, _, _ = sets[i]
                o = ops.block_attention(q, k, v, blocks)
                got[i].append((o.detach(),) + torch.autograd.grad(o, (q, k, v), go)
                              + (ops.sparse_attention(q[:, :1].detach(), k.detach(), v.detach(), 3),))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, c) for a, c in zip(r, want[i] + (few[i],)))


@pytest.mark.parametrize("n", [200, 2100])
def test_captured_and_replayed(dev, n):
    """norm_rotate, selection, attention and their gradients in one graph; replayed with other inputs and the program's own
    eager calls in between, two graphs of the same operators at once."""
    ops = pkg("network.operations")
    freq = ops.rotation_frequencies(1, 16, device=dev)
    position = torch.arange(n, device=dev).expand(2, n)

    def make(seed):
        gen = _gen(dev, seed)
        return [_randn(gen, 2, n, h, 32, dtype=torch.float16) for h in (4, 2, 2)] + [1 + 0.1 * _randn(gen, 32), _randn(gen, 2, n, 4, 32, dtype=torch.float16)]

    def step(q, k, v, w, go):
        q, k, v, w = (t.detach().requires_grad_() for t in (q, k, v, w))
        a, c = ops.norm_rotate(q, k, w, w, position, freq)
        o = ops.sparse_attention(a, c, v, 2, causal=True)
        few = ops.sparse_attention(a[:, -1:].detach(), c.detach(), v.detach(), 2, causal=True)
        return (o.detach(), few) + torch.autograd.grad(o, (q, k, v, w), go)

    graphs = []
    for seed in (1, 2):
        held = make(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held)
        graphs.append((held, graph, out))
    for seed in range(10, 14):
        for held, graph, out in graphs:
            new = make(seed)
            for t, x in zip(held, new):
                t.copy_(x)
        for held, graph, out in graphs:
            graph.replay()
        want = step(*make(seed))
        torch.cuda.synchronize()
        for held, graph, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_backward_twice_and_changed_inputs(dev):
    ops = pkg("network.operations")
    q, k, v, go, blocks, _, _ = _attend_inputs(dev, (1, 30, 100, 2, 1, 16, 2, False, False), torch.float32, 7)
    q.requires_grad_()
    o = ops.block_attention(q, k, v, blocks)
    a, = torch.autograd.grad(o, q, go, retain_graph=True)
    c, = torch.autograd.grad(o, q, go, retain_graph=True)
    assert torch.equal(a, c)
    k += 1                                                                  # saved for the backward pass
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, q, go)
    # gradients of gradients are not offered
    o = ops.block_attention(q, k, v, blocks)
    d, = torch.autograd.grad(o, q, go.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), q)


def test_refusals(dev):
    ops = pkg("network.operations")
    x = torch.zeros((1, 4, 2, 16), device=dev)
    pos, freq = torch.zeros((1, 4), device=dev), ops.rotation_frequencies(1, 8, device=dev)
    bad = [
        lambda: ops.norm_rotate(x[0], None, None, None, pos, freq),
        lambda: ops.norm_rotate(x.double(), None, None, None, pos, freq),
        lambda: ops.norm_rotate(torch.zeros((1, 4, 2, 12), device=dev), None, None, None, pos, freq),
        lambda: ops.norm_rotate(torch.zeros((1, 4, 2, 264), device=dev), None, None, None, pos, freq),
        lambda: ops.norm_rotate(x, x.half(), None, None, pos, freq),
        lambda: ops.norm_rotate(x, x[:, :3], None, None, pos, freq),
        lambda: ops.norm_rotate(x, None, None, torch.ones(16, device=dev), pos, freq),
        lambda: ops.norm_rotate(x, None, torch.ones(8, device=dev), None, pos, freq),
        lambda: ops.norm_rotate(x, None, torch.ones(16), None, pos, freq),
        lambda: ops.norm_rotate(x, None, None, None, pos[:, :3], freq),
        lambda: ops.norm_rotate(x, None, None, None, pos.half(), freq),
        lambda: ops.norm_rotate(x, None, None, None, pos.requires_grad_(), freq),
        lambda: ops.norm_rotate(x, None, None, None, pos.detach(), ops.rotation_frequencies(1, 9, device=dev)),
        lambda: ops.norm_rotate(x, None, None, None, pos.detach(), ops.rotation_frequencies(2, 2, device=dev)),
        lambda: ops.norm_rotate(x, None, None, None, pos.detach(), freq, eps=-1.0),
        lambda: ops.norm_rotate(torch.zeros((1, 4, 200, 128), device=dev), None, torch.ones((200, 128), device=dev, requires_grad=True),
                                None, pos.detach(), freq),
    ]
    k = torch.zeros((1, 130, 1, 16), device=dev)
    blocks = torch.zeros((1, 4, 1, 2), dtype=torch.int32, device=dev)
    means = ops.block_means(k)
    bad += [
        lambda: ops.block_means(k, last=1),
        lambda: ops.block_means(k, out=means, last=-1),
        lambda: ops.block_means(k, out=means[:, :2]),
        lambda: ops.block_means(torch.zeros((1, 4, 1, 136), device=dev)),
        lambda: ops.block_means(k, torch.zeros(2, dtype=torch.int32, device=dev)),
        lambda: ops.block_means(k, torch.zeros(1, dtype=torch.int64, device=dev)),
        lambda: ops.select_blocks(x, means, 130, 0),
        lambda: ops.select_blocks(x, means, 130, 65),
        lambda: ops.select_blocks(x, means, 200, 2),
        lambda: ops.select_blocks(x, means.half(), 130, 2),
        lambda: ops.select_blocks(x, torch.zeros((1, 3, 0, 16), device=dev), 130, 2),
        lambda: ops.block_attention(x, k, k[:, :129], blocks),
        lambda: ops.block_attention(x, k.half(), k.half(), blocks),
        lambda: ops.block_attention(x, k, k, blocks[:, :3]),
        lambda: ops.block_attention(x, k, k, blocks.float()),
        lambda: ops.block_attention(x, k, k, blocks.cpu()),
        lambda: ops.block_attention(x, k, k, blocks, scale=0.0),
        lambda: ops.block_attention(x, k, k, blocks, scale=math.inf),
        lambda: ops.block_attention(x, k, k, blocks, scale=math.nan),
        lambda: ops.block_attention(torch.zeros((1, 4, 65, 16), device=dev), k, k, blocks),
        lambda: ops.block_attention(torch.zeros((1, 4, 3, 16), device=dev), torch.zeros((1, 9, 2, 16), device=dev),
                                    torch.zeros((1, 9, 2, 16), device=dev), blocks),
        lambda: ops.sparse_attention(x, k, k, 2, means=means[:, :1]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            print("call %d was taken" % i)
