"""Attention between points: the learned form of what the inter-level skip does with a fixed kernel (reference
network/upsampler.py:317-347: a cheap search picks rows of another point set, their weights are normalised, the rows are
added up).  The reference has no such operator.  Public through `network.operations`.

    q, k = norm_rotate(q, k, q_weight, k_weight, position, freq)     per-head norms, rotation by the position
    o = sparse_attention(q, k, v, count)                             = the three below in a row
        means  = block_means(k)                                      mean of every block of 64 consecutive keys
        blocks = select_blocks(q, means, k.size(1), count)           the `count` best blocks of every query
        o      = block_attention(q, k, v, blocks)                    softmax attention over their keys

Tensors are channel-last with a head axis, (B, rows, heads, D), float32, float16 or bfloat16, D a multiple of 8; any strides
(what is not 16-byte rows with unit channel stride is copied).  Keys may have fewer heads than queries (a group of query
heads shares a key head and its blocks).  n_arr / m_arr: int32 device tensors of the live keys / queries of each sequence, as
in the ragged point-set calls.  causal: query i stands at key position n - m + i (live lengths) and sees the keys up to it.
Rows near each other should hold points near each other (a space-filling order, a sequence): a block is then a neighbourhood.

Gradients are those of reverse mode, once; where there are any, an input with a tangent of forward mode is refused.  Device
tensors only; everything runs on the current stream of the tensors' device and can be captured into a graph (a backward
pass: torch.autograd.grad, or backward() while no eager graph of the same leaves is alive, which torch itself cannot capture).
Results do not depend on the order in which workgroups run.

A key, query, value or output gradient that is not finite reaches what its masks let it reach and nothing else; a gradient that
it reaches is not a number as a whole row.  Scores, softmax statistics, sums and norms are held in 32 bits or more; the 16-bit
types take probabilities and score gradients into the second matrix products in two terms of their own type, which together hold
2^-17 (bfloat16) or 2^-22 (float16) of a value; float32 rounds nothing.  Means of blocks and scores of blocks are formed in 64 bits."""
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib as L

BLOCK = L.ATTN_BLOCK        # consecutive keys of a block


def _rows(t, name, like=None):
    """The checks of a (B, rows, heads, D) tensor."""
    if isinstance(t, torch.Tensor) and t.dim() and max(t.shape) > 0x7FFFFFFF:
        raise RuntimeError("%s: dimensions of at most 2^31 - 1, got %s" % (name, tuple(t.shape)))
    if not isinstance(t, torch.Tensor) or t.get_device() < 0:
        raise RuntimeError("%s must be a CUDA tensor" % name)
    if t.dim() != 4:
        raise RuntimeError("%s must be (B, rows, heads, D), got %s" % (name, tuple(t.shape)))
    if t.dtype not in L.TYPES:
        raise RuntimeError("%s must be float32, float16 or bfloat16, got %s" % (name, t.dtype))
    if like is not None and (t.dtype != like.dtype or t.get_device() != like.get_device()):
        raise RuntimeError("%s must be %s on %s, got %s on %s" % (name, like.dtype, like.device, t.dtype, t.device))
    d = t.shape[3]
    if d == 0 or d % 8:
        raise RuntimeError("%s: D must be a multiple of 8, got %d" % (name, d))
    return t


def _no_tangents(*tensors):
    """There is no forward-mode derivative: the kernels' results would carry none, which means 0."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return                                          # (no dual level is open: no tensor has a tangent)
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("forward-mode derivatives are not offered: an input carries a tangent")


def _taken(t):
    if t is None or (t.is_contiguous() and not t.data_ptr() & 15):
        return t                                        # (rows of a multiple of 8 channels: 16 bytes)
    per = 16 // t.element_size()
    if t.stride(3) != 1 or t.data_ptr() & 15 or any(t.size(i) > 1 and t.stride(i) % per for i in range(3)):
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
    return t


_ABSENT = L.Heads(None, 0, 0, 0, 0)


def _heads(t):
    """tpu3_heads of a tensor that _taken returned; None: absent."""
    if t is None:
        return _ABSENT
    size, stride = t.shape, t.stride()
    return L.Heads(t.data_ptr() or None, stride[0] if size[0] > 1 else 0, stride[1] if size[1] > 1 else 0,
                   stride[2] if size[2] > 1 else 0, size[2])


# the stream handle without the Stream object around it (2 us of a call's 10)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _launch(name, t, *args):
    """A C entry point on the current stream of the tensor's device (which is made the current device if it is not)."""
    dev = t.get_device()
    if torch.cuda.current_device() == dev:
        rc = getattr(L.lib(), name)(_raw_stream(dev), *args)
    else:
        with torch.cuda.device(dev):
            rc = getattr(L.lib(), name)(_raw_stream(dev), *args)
    if rc:
        L.check(rc, name)


def _workspace(need, t):
    return t.new_empty((need,), dtype=torch.uint8) if need else None


def _lengths(t, name, b, like):
    if t is None:
        return None
    L.require_device(t, name)
    L.require_dtype(t, torch.int32, name)
    if t.shape != (b,) or t.get_device() != like.get_device():
        raise RuntimeError("%s must be (%d,) on %s, got %s on %s" % (name, b, like.device, tuple(t.shape), t.device))
    return t


# ---- norms and rotation ------------------------------------------------------------------------------------------------
def rotation_frequencies(axes, pairs, base=10000.0, device=None):
    """(axes, pairs) float64: base ** (-f / pairs) for every axis, the frequencies of a position in a sequence."""
    f = float(base) ** (-torch.arange(pairs, dtype=torch.float64, device=device) / max(1, pairs))
    return f.repeat(axes, 1)


def _rotation(q, position, freq):
    s = position.stride()
    return L.Positions(position.data_ptr(), s[0], s[1], s[2], L.POSITION_TYPES[position.dtype], freq.size(0), freq.size(1),
                       freq.data_ptr() or None, L.POSITION_TYPES[freq.dtype])


def _weights(wq, wk, d):
    some = wq if wq is not None else wk
    return (L.ptr(wq), d if wq is not None and wq.dim() == 2 else 0, L.ptr(wk), d if wk is not None and wk.dim() == 2 else 0,
            L.TYPES[some.dtype] if some is not None else 0)


def _norm_rotate_forward(q, k, wq, wk, position, freq, eps, interleaved):
    q, k = _taken(q), _taken(k)
    oq = q.new_empty(q.shape)
    ok = None if k is None else k.new_empty(k.shape)
    b, n, _, d = q.shape
    _launch("tpu3_norm_rotate_fwd", q, L.TYPES[q.dtype], b, n, d, _heads(q), _heads(k), *_weights(wq, wk, d),
            _rotation(q, position, freq), eps, interleaved, oq.data_ptr(), L.ptr(ok))
    return oq, ok


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, position, freq, eps, interleaved):
        ctx.save_for_backward(q, k, wq, wk, position, freq)
        ctx.eps, ctx.interleaved = eps, interleaved
        return _norm_rotate_forward(q, k, wq, wk, position, freq, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        _no_tangents(gq, gk)
        q, k, wq, wk, position, freq = ctx.saved_tensors
        q, k, gq = _taken(q), _taken(k), _taken(gq)
        gk = None if k is None else _taken(gk)
        b, n, hq, d = q.shape
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
        make = torch.zeros if b * n == 0 else torch.empty            # (no rows: the kernels do not run)
        dwq, dwk = (make(w.shape, dtype=w.dtype, device=w.device) if w is not None and need else None
                    for w, need in ((wq, ctx.needs_input_grad[2]), (wk, ctx.needs_input_grad[3])))
        need = 0
        if dwq is not None or dwk is not None:
            per_head = int((wq if wq is not None else wk).dim() == 2)
            need = L.lib().tpu3_norm_rotate_bwd_workspace_bytes(hq + (0 if k is None else k.size(2)), d, per_head)
        ws = _workspace(need, q)
        _launch("tpu3_norm_rotate_bwd", q, L.TYPES[q.dtype], b, n, d, _heads(q), _heads(k), *_weights(wq, wk, d),
                _rotation(q, position, freq), ctx.eps, ctx.interleaved, _heads(gq), _heads(gk), dq.data_ptr(), L.ptr(dk),
                L.ptr(dwq), L.ptr(dwk), L.ptr(ws), need)
        return dq, dk, dwq, dwk, None, None, None, None


def norm_rotate(q, k, q_weight, k_weight, position, freq, eps=1e-6, interleaved=False):
    """Norm of every head's row and its rotation by the row's position, queries and keys in one launch.
    :param
        q         (B, N, Hq, D); D <= 256
        k         (B, N, Hk, D) or None
        q_weight, k_weight  (D,) for all heads, (heads, D), or None for ones; (heads, D) with a gradient: (Hq + Hk) * D at
                  most 24576
        position  (B, N) or (B, N, axes): places in a sequence (int32 / int64) or coordinates (float32 / float64)
        freq      (axes, pairs) float32 / float64, 2 * axes * pairs <= D: pair axis * pairs + f turns by
                  position[axis] * freq[axis, f], an angle formed in 64 bits
        eps       y = x / sqrt(mean(x^2) + eps) * weight, the mean in float32: rows with elements beyond 1e19 come out as 0
        interleaved   partners of pair p are channels (2p, 2p + 1) instead of (p, p + axes * pairs)
    :return
        (q, k) of the inputs' shapes and types (k None if it was None)
    Differentiable in q, k and the weights; position and freq are constants (refused if they require a gradient)."""
    q = _rows(q, "q")
    b, n, hq, d = q.shape
    if d > 256:
        raise RuntimeError("norm_rotate: D must be at most 256, got %d" % d)
    if k is not None:
        k = _rows(k, "k", q)
        if (k.size(0), k.size(1), k.size(3)) != (b, n, d):
            raise RuntimeError("norm_rotate: q %s and k %s do not match" % (tuple(q.shape), tuple(k.shape)))
    elif k_weight is not None:
        raise RuntimeError("norm_rotate: k_weight without k")
    if hq == 0 or (k is not None and k.size(2) == 0) or max(hq, 0 if k is None else k.size(2)) > 1024:
        raise RuntimeError("norm_rotate: 1 to 1024 heads")
    weights = []
    for w, h, name in ((q_weight, hq, "q_weight"), (k_weight, 0 if k is None else k.size(2), "k_weight")):
        if w is not None:
            if w.get_device() != q.get_device():
                raise RuntimeError("%s must be a CUDA tensor on %s" % (name, q.device))
            if w.dtype not in L.TYPES:
                raise RuntimeError("%s must be float32, float16 or bfloat16, got %s" % (name, w.dtype))
            if w.shape != (d,) and w.shape != (h, d):
                raise RuntimeError("%s must be (%d,) or (%d, %d), got %s" % (name, d, h, d, tuple(w.shape)))
        weights.append(w)
    wq, wk = weights
    if wq is not None and wk is not None:
        if wq.dtype != wk.dtype or wq.dim() != wk.dim():
            wq, wk = wq.float(), wk.float()              # (32 bits: the heads' gradients of a shared set are added up)
        if wq.dim() != wk.dim():
            wq, wk = wq.expand(hq, d), wk.expand(k.size(2), d)
    wq, wk = (w if w is None or (w.is_contiguous() and not w.data_ptr() & 15) else w.contiguous().clone() for w in (wq, wk))
    if position.get_device() != q.get_device() or freq.get_device() != q.get_device():
        raise RuntimeError("position and freq must be CUDA tensors on %s" % q.device)
    if position.dtype not in L.POSITION_TYPES:
        raise RuntimeError("position must be float32, float64, int32 or int64, got %s" % position.dtype)
    if freq.dtype not in (torch.float32, torch.float64):
        raise RuntimeError("freq must be float32 or float64, got %s" % freq.dtype)
    if position.requires_grad or freq.requires_grad:
        raise RuntimeError("norm_rotate: position and freq are constants: pass them detached")
    if position.dim() == 2:
        position = position.unsqueeze(2)
    if position.dim() != 3 or freq.dim() != 2 or position.shape != (b, n, freq.shape[0]) or freq.shape[0] == 0:
        raise RuntimeError("norm_rotate: position %s and freq %s do not fit %d x %d rows"
                           % (tuple(position.shape), tuple(freq.shape), b, n))
    _no_tangents(q, k, q_weight, k_weight, position, freq)
    if 2 * freq.numel() > d:
        raise RuntimeError("norm_rotate: %d pairs need more than %d channels" % (freq.numel(), d))
    args = (q, k, wq, wk, position, freq.contiguous(), float(eps), int(bool(interleaved)))
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:4])
    if grad and any(w is not None and w.dim() == 2 and w.requires_grad for w in (wq, wk)) \
            and (hq + (0 if k is None else k.size(2))) * d > 24576:
        raise RuntimeError("norm_rotate: the gradient of weights for every head needs heads * D of at most 24576")
    return _NormRotate.apply(*args) if grad else _norm_rotate_forward(*args)


# ---- blocks ------------------------------------------------------------------------------------------------------------
def _count(count):
    if not 1 <= int(count) <= L.BLOCK_COUNT_MAX:
        raise RuntimeError("count must be 1 to %d, got %s" % (L.BLOCK_COUNT_MAX, count))
    return int(count)


def _keys(keys):
    if (keys + BLOCK - 1) // BLOCK > L.ATTN_BLOCKS_MAX:
        raise RuntimeError("at most %d keys, got %d" % (BLOCK * L.ATTN_BLOCKS_MAX, keys))
    return keys


def block_means(k, n_arr=None, out=None, last=None):
    """Means of the blocks of 64 consecutive keys, the summary that select_blocks scores.
    :param
        k       (B, N, Hk, D); D <= 128
        n_arr   live keys of each sequence
        out     (B, ceil(N / 64), Hk, D) float32 contiguous to write to
        last    with `out`: only the blocks that hold the last `last` live keys are formed again (keys were appended), the
                others are left as they are
    :return
        (B, ceil(N / 64), Hk, D) float32, summed in 64 bits and rounded once; a block without a live key: 0.  No gradient."""
    k = _rows(k.detach() if isinstance(k, torch.Tensor) else k, "k")
    b, n, hk, d = k.shape
    if d > 128:
        raise RuntimeError("block_means: D must be at most 128, got %d" % d)
    if hk == 0:
        raise RuntimeError("block_means: k has no heads")
    n_arr = _lengths(n_arr, "n_arr", b, k)
    shape = (b, (_keys(n) + BLOCK - 1) // BLOCK, hk, d)
    if out is None:
        if last is not None:
            raise RuntimeError("block_means: last without out")
        out = torch.empty(shape, dtype=torch.float32, device=k.device)
    else:
        L.require_device(out, "out")
        L.require_dtype(out, torch.float32, "out")
        if tuple(out.shape) != shape or out.device != k.device or out.requires_grad or out.data_ptr() & 15:
            raise RuntimeError("out must be %s on %s, 16-byte aligned, without a gradient" % (shape, k.device))
    if last is not None and int(last) < 0:
        raise RuntimeError("block_means: last must not be negative, got %s" % last)
    k = _taken(k)
    _launch("tpu3_block_means", k, L.TYPES[k.dtype], b, n, d, _heads(k), L.ptr(n_arr),
            -1 if last is None else min(int(last), n), out.data_ptr())
    return out


def select_blocks(q, means, keys, count, n_arr=None, m_arr=None, causal=False):
    """The blocks of keys that every query attends to.
    :param
        q       (B, M, Hq, D)
        means   (B, ceil(keys / 64), Hk, D) float32 of block_means; Hq a multiple of Hk
        keys    number of keys (N of the key tensor)
        count   blocks a query and key head, 1 to 64
    :return
        (B, M, Hk, count) int32, ascending, -1 behind the found ones.  The best `count` of (sum of the group's query
        rows) . mean, scored in 64 bits, equal ones to the lowest block, a score that is not a number last; causal: the block of the query's own position
        always, the others among those before it.  Queries behind m_arr: all -1.  No gradient."""
    q = _rows(q.detach() if isinstance(q, torch.Tensor) else q, "q")
    b, m, hq, d = q.shape
    count, keys = _count(count), _keys(int(keys))
    if not isinstance(means, torch.Tensor) or means.get_device() < 0:
        raise RuntimeError("means must be a CUDA tensor")
    L.require_dtype(means, torch.float32, "means")
    if means.dim() != 4 or (means.size(0), means.size(1), means.size(3)) != (b, (keys + BLOCK - 1) // BLOCK, d) \
            or means.get_device() != q.get_device():
        raise RuntimeError("means %s do not fit q %s and %d keys" % (tuple(means.shape), tuple(q.shape), keys))
    hk = means.size(2)
    if hk == 0 or hq == 0 or hq % hk:
        raise RuntimeError("select_blocks: %d query heads over %d key heads" % (hq, hk))
    if d > 128:
        raise RuntimeError("select_blocks: D must be at most 128, got %d" % d)
    n_arr, m_arr = _lengths(n_arr, "n_arr", b, q), _lengths(m_arr, "m_arr", b, q)
    means = means.detach().contiguous()
    if means.data_ptr() & 15:
        means = means.clone()
    blocks = q.new_empty((b, m, hk, count), dtype=torch.int32)
    q = _taken(q)
    need = L.lib().tpu3_block_select_workspace_bytes(b, m, keys, hk, count)
    ws = _workspace(need, q)
    _launch("tpu3_block_select", q, L.TYPES[q.dtype], b, m, keys, d, _heads(q), hk, means.data_ptr(), L.ptr(n_arr),
            L.ptr(m_arr), int(bool(causal)), count, blocks.data_ptr(), L.ptr(ws), need)
    return blocks


def _attention_forward(q, k, v, blocks, scale, n_arr, m_arr, causal, grad=False):
    """-> o, and for the backward pass lse and what the rounding of a 16-bit o took (else None)."""
    q, k, v = _taken(q), _taken(k), _taken(v)
    b, m, hq, d = q.shape
    n, hk, count = k.size(1), k.size(2), blocks.size(3)
    o = q.new_empty(q.shape)
    lse = q.new_empty((b, hq, m, 2), dtype=torch.float32) if grad else None
    rest = q.new_empty(q.shape) if grad and q.dtype != torch.float32 else None
    need = L.lib().tpu3_block_attn_fwd_workspace_bytes(b, m, n, hq, hk, d, count)
    ws = _workspace(need, q)
    _launch("tpu3_block_attn_fwd", q, L.TYPES[q.dtype], b, m, n, d, _heads(q), _heads(k), _heads(v), blocks.data_ptr(), count,
            scale, L.ptr(n_arr), L.ptr(m_arr), causal, o.data_ptr(), L.ptr(lse), L.ptr(rest), L.ptr(ws), need)
    return o, lse, rest


class _BlockAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, blocks, scale, n_arr, m_arr, causal):
        o, lse, rest = _attention_forward(q, k, v, blocks, scale, n_arr, m_arr, causal, True)
        ctx.save_for_backward(q, k, v, o, lse, rest, blocks, n_arr, m_arr)
        ctx.scale, ctx.causal = scale, causal
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        _no_tangents(go)
        q, k, v, o, lse, rest, blocks, n_arr, m_arr = ctx.saved_tensors
        q, k, v, o, go = (_taken(t) for t in (q, k, v, o, go))
        b, m, hq, d = q.shape
        n, hk, count = k.size(1), k.size(2), blocks.size(3)
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        make = torch.zeros if m == 0 else torch.empty                # (no queries: the kernels do not run)
        dk, dv = (make(t.shape, dtype=t.dtype, device=t.device) for t in (k, v))
        need = L.lib().tpu3_block_attn_bwd_workspace_bytes(b, m, n, hq, hk, d, count)
        ws = _workspace(need, q)
        _launch("tpu3_block_attn_bwd", q, L.TYPES[q.dtype], b, m, n, d, _heads(q), _heads(k), _heads(v), _heads(o), _heads(go),
                blocks.data_ptr(), count, ctx.scale, L.ptr(n_arr), L.ptr(m_arr), ctx.causal, lse.data_ptr(), L.ptr(rest),
                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), L.ptr(ws), need)
        return dq, dk, dv, None, None, None, None, None


def _attention(q, k, v, *args):
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _BlockAttention.apply(q, k, v, *args)
    return _attention_forward(q, k, v, *args)[0]


def _check_attention(q, k, v, scale, n_arr, m_arr):
    q = _rows(q, "q")
    k, v = _rows(k, "k", q), _rows(v, "v", q)
    _no_tangents(q, k, v)
    b, m, hq, d = q.shape
    if v.shape != k.shape or k.shape[0] != b or k.shape[3] != d:
        raise RuntimeError("q %s, k %s and v %s do not match" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    hk = k.size(2)
    if hk == 0 or hq == 0 or hq % hk or hq // hk > 64:
        raise RuntimeError("%d query heads over %d key heads: a group of 1 to 64" % (hq, hk))
    if d > 128:
        raise RuntimeError("D must be at most 128, got %d" % d)
    _keys(k.size(1))
    scale = d ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise RuntimeError("scale must be 1e-30 to 1e30, got %s" % scale)
    return q, k, v, scale, _lengths(n_arr, "n_arr", b, q), _lengths(m_arr, "m_arr", b, q)


def block_attention(q, k, v, blocks, scale=None, n_arr=None, m_arr=None, causal=False):
    """Softmax attention of every query over the keys of the blocks named for it.
    :param
        q       (B, M, Hq, D); D <= 128
        k, v    (B, N, Hk, D); Hq a multiple of Hk, at most 64 query heads a key head
        blocks  (B, M, Hk, count) int32 / int64, count <= 64: blocks of 64 consecutive keys, in any order; an index outside
                the live blocks, or behind what a causal query sees, counts for nothing, one named twice counts once
        scale   factor of the scores, positive (default D ** -0.5)
    :return
        (B, M, Hq, D) of q's type; a row that sees nothing (or is behind m_arr): 0
    Differentiable in q, k and v (keys behind n_arr: gradient 0)."""
    q, k, v, scale, n_arr, m_arr = _check_attention(q, k, v, scale, n_arr, m_arr)
    if not isinstance(blocks, torch.Tensor) or blocks.get_device() != q.get_device():
        raise RuntimeError("blocks must be a CUDA tensor on %s" % q.device)
    if blocks.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("blocks must be int32 or int64, got %s" % blocks.dtype)
    if blocks.dim() != 4 or tuple(blocks.shape[:3]) != (q.size(0), q.size(1), k.size(2)):
        raise RuntimeError("blocks %s do not fit q %s and %d key heads" % (tuple(blocks.shape), tuple(q.shape), k.size(2)))
    _count(blocks.size(3))
    if blocks.dtype == torch.int64:
        blocks = blocks.clamp(-1, L.ATTN_BLOCKS_MAX).to(torch.int32)
    return _attention(q, k, v, blocks.contiguous(), scale, n_arr, m_arr, int(bool(causal)))


def sparse_attention(q, k, v, count, scale=None, n_arr=None, m_arr=None, causal=False, means=None):
    """block_attention over the `count` blocks that select_blocks picks for every query.  `means`: those of block_means for
    these keys, where a program keeps them (a cache that grows: block_means(..., out=means, last=appended)); formed here if
    not given.  Differentiable in q, k and v; which blocks are read is a constant of the step."""
    q, k, v, scale, n_arr, m_arr = _check_attention(q, k, v, scale, n_arr, m_arr)
    if means is None:
        means = block_means(k, n_arr)
    blocks = select_blocks(q, means, k.size(1), count, n_arr, m_arr, causal)
    if means.size(2) != k.size(2):
        raise RuntimeError("means have %d heads, k has %d" % (means.size(2), k.size(2)))
    return _attention(q, k, v, blocks, scale, n_arr, m_arr, int(bool(causal)))
