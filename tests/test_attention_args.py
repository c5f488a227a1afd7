"""What the attention entry points refuse before they launch anything: the C functions with arguments out of range (a status,
no launch), the Python functions with tensors that are not on a GPU."""
import pytest
import torch

from conftest import pkg

EINVAL, ELIMIT = -1, -2


@pytest.fixture(scope="module")
def abi():
    return pkg("_lib")


def _heads(L, heads=2, data=1 << 20, sb=0, sr=256, sh=64):
    return L.Heads(data, sb, sr, sh, heads)


def _positions(L, axes=1, pairs=8, kind=0, freq=0):
    return L.Positions(1 << 20, 0, 1, 0, kind, axes, pairs, 1 << 20, freq)


def test_workspace_sizes(abi):
    lib = abi.lib()
    assert lib.tpu3_block_select_workspace_bytes(0, 5, 100, 1, 4) == 0
    assert lib.tpu3_block_select_workspace_bytes(1, 5, 0, 1, 4) == 0
    assert lib.tpu3_block_select_workspace_bytes(1, 5, 100, 1, 65) == 0
    assert lib.tpu3_block_select_workspace_bytes(2, 4096, 4096, 8, 16) == 2 * 8 * 64 * 8         # a word a 64 queries
    assert lib.tpu3_block_select_workspace_bytes(1, 1, 64 * 256, 1, 16) == 0
    assert lib.tpu3_block_select_workspace_bytes(1, 1, 64 * 640, 1, 16) == 5 * 16 * 12           # five parts of 128 blocks
    assert lib.tpu3_block_attn_fwd_workspace_bytes(4, 4096, 4096, 8, 8, 64, 16) == 0
    one = lib.tpu3_block_attn_fwd_workspace_bytes(1, 1, 4096, 8, 2, 128, 16)
    assert one > 0 and one % (8 * (128 + 4) * 4) == 0
    assert lib.tpu3_block_attn_fwd_workspace_bytes(1, 0, 4096, 8, 2, 128, 16) == 0
    assert lib.tpu3_block_attn_bwd_workspace_bytes(1, 0, 4096, 8, 2, 128, 16) == 0
    # bits, do . o and the largest |do| of every row, a flag; no parts where there are more than 1024 blocks
    rows = (2 * 8 * 4096 * 4 + 15) // 16 * 16
    assert lib.tpu3_block_attn_bwd_workspace_bytes(2, 4096, 64 * 65, 8, 8, 64, 16) == 2 * 8 * 65 * 64 * 8 + 2 * rows + 16
    assert lib.tpu3_norm_rotate_bwd_workspace_bytes(0, 64, 1) == 0
    assert lib.tpu3_norm_rotate_bwd_workspace_bytes(6, 64, 1) == 3 * lib.tpu3_norm_rotate_bwd_workspace_bytes(6, 64, 0)


NORM = [
    (dict(type=7), EINVAL), (dict(b=-1), EINVAL), (dict(n=-1), EINVAL), (dict(d=0), EINVAL), (dict(d=12), ELIMIT),
    (dict(d=264), ELIMIT), (dict(eps=-1.0), EINVAL), (dict(eps=float("nan")), EINVAL), (dict(wq_head=8), EINVAL),
    (dict(q=dict(data=0)), EINVAL), (dict(q=dict(data=(1 << 20) + 2)), EINVAL), (dict(q=dict(sr=3)), EINVAL),
    (dict(q=dict(heads=0)), EINVAL), (dict(q=dict(heads=1025)), ELIMIT), (dict(k=dict(heads=1025)), ELIMIT),
    (dict(k=dict(heads=-1)), EINVAL), (dict(k=dict(sh=1)), EINVAL), (dict(pos=dict(axes=0)), EINVAL), (dict(pos=dict(pairs=9)), EINVAL),
    (dict(pos=dict(axes=2)), EINVAL), (dict(pos=dict(kind=9)), EINVAL), (dict(pos=dict(freq=2)), EINVAL), (dict(oq=0), EINVAL),
    (dict(oq=8), EINVAL), (dict(ok=0), EINVAL), (dict(wq=8), EINVAL), (dict(w_type=5), EINVAL), (dict(n=0), 0), (dict(b=0), 0),
]


@pytest.mark.parametrize("change,want", NORM)
def test_norm_rotate_status(abi, change, want):
    c = dict(type=0, b=1, n=4, d=16, wq=0, wq_head=0, w_type=0, eps=1e-6, oq=1 << 20, ok=1 << 20, q={}, k={}, pos={})
    c.update(change)
    q, k, pos = _heads(abi, **c["q"]), _heads(abi, **c["k"]), _positions(abi, **c["pos"])
    args = (None, c["type"], c["b"], c["n"], c["d"], q, k, c["wq"], c["wq_head"], None, 0, c["w_type"], pos, c["eps"], 0)
    assert abi.lib().tpu3_norm_rotate_fwd(*args, c["oq"], c["ok"]) == want
    if "oq" in change or "ok" in change:
        return
    assert abi.lib().tpu3_norm_rotate_bwd(*args, q, k, 1 << 20, 1 << 20, None, None, None, 0) == want


def test_norm_rotate_backward_status(abi):
    q = _heads(abi)
    args = (None, 0, 1, 4, 16, q, q, 1 << 20, 0, None, 0, 0, _positions(abi), 1e-6, 0)
    f = abi.lib().tpu3_norm_rotate_bwd
    assert f(*args, q, q, 1 << 20, 1 << 20, 1 << 20, None, None, 0) == EINVAL                    # a weight gradient, no workspace
    assert f(*args, q, q, 1 << 20, 1 << 20, 1 << 20, None, 1 << 20, 64) == EINVAL
    assert f(*args, _heads(abi, heads=3), q, 1 << 20, 1 << 20, None, None, None, 0) == EINVAL
    assert f(*args, q, q, 0, 1 << 20, None, None, None, 0) == EINVAL
    assert f(*args, q, q, 1 << 20, 0, None, None, None, 0) == EINVAL


MEANS = [
    (dict(type=3), EINVAL), (dict(b=-1), EINVAL), (dict(n=-2), EINVAL), (dict(d=0), EINVAL), (dict(d=136), ELIMIT), (dict(d=20), ELIMIT),
    (dict(k=dict(heads=0)), EINVAL), (dict(k=dict(data=0)), EINVAL), (dict(k=dict(sb=2)), EINVAL), (dict(means=0), EINVAL),
    (dict(means=4), EINVAL), (dict(b=0), 0), (dict(n=0), 0), (dict(last=0), 0), (dict(b=1 << 16, n=1 << 30), ELIMIT),
]


@pytest.mark.parametrize("change,want", MEANS)
def test_block_means_status(abi, change, want):
    c = dict(type=0, b=1, n=100, d=16, k={}, last=-1, means=1 << 20)
    c.update(change)
    assert abi.lib().tpu3_block_means(None, c["type"], c["b"], c["n"], c["d"], _heads(abi, **c["k"]), None, c["last"], c["means"]) == want


SELECT = [
    (dict(type=-1), EINVAL), (dict(b=-1), EINVAL), (dict(m=-1), EINVAL), (dict(n=-1), EINVAL), (dict(d=0), EINVAL), (dict(hk=0), EINVAL),
    (dict(hk=3), EINVAL), (dict(count=0), EINVAL), (dict(count=65), ELIMIT), (dict(d=136), ELIMIT), (dict(n=2**31 - 1), ELIMIT),
    (dict(q=dict(data=0)), EINVAL), (dict(q=dict(sr=2)), EINVAL), (dict(means=0), EINVAL), (dict(means=8), EINVAL), (dict(blocks=0), EINVAL),
    (dict(m=5000), EINVAL), (dict(n=64 * 640), EINVAL), (dict(m=0), 0), (dict(b=0), 0),
]


@pytest.mark.parametrize("change,want", SELECT)
def test_block_select_status(abi, change, want):
    c = dict(type=0, b=1, m=5, n=100, d=16, q={}, hk=2, means=1 << 20, count=4, blocks=1 << 20)
    c.update(change)
    # (no workspace: where the call needs one, it is refused)
    assert abi.lib().tpu3_block_select(None, c["type"], c["b"], c["m"], c["n"], c["d"], _heads(abi, **c["q"]), c["hk"], c["means"],
                                       None, None, 0, c["count"], c["blocks"], None, 0) == want


ATTEND = [
    (dict(type=9), EINVAL), (dict(b=-1), EINVAL), (dict(m=-1), EINVAL), (dict(n=-1), EINVAL), (dict(d=-8), EINVAL), (dict(d=9), ELIMIT),
    (dict(d=136), ELIMIT), (dict(count=0), EINVAL), (dict(count=65), ELIMIT), (dict(n=2**31 - 1), ELIMIT), (dict(q=dict(heads=3)), EINVAL),
    (dict(q=dict(heads=130)), ELIMIT), (dict(k=dict(heads=0)), EINVAL), (dict(v=dict(heads=1)), EINVAL), (dict(q=dict(data=0)), EINVAL),
    (dict(k=dict(data=0)), EINVAL), (dict(v=dict(data=8)), EINVAL), (dict(v=dict(sr=6)), EINVAL), (dict(scale=0.0), EINVAL),
    (dict(scale=-1.0), EINVAL), (dict(scale=float("nan")), EINVAL), (dict(scale=float("inf")), EINVAL), (dict(blocks=0), EINVAL),
    (dict(out=0), EINVAL), (dict(out=8), EINVAL), (dict(rest=4), EINVAL), (dict(m=0), 0), (dict(b=0), 0),
]


@pytest.mark.parametrize("change,want", ATTEND)
def test_block_attention_status(abi, change, want):
    c = dict(type=0, b=1, m=5, n=40, d=16, q={}, k={}, v={}, blocks=1 << 20, count=4, scale=0.25, out=1 << 20, rest=0)
    c.update(change)
    q, k, v = (_heads(abi, **c[x]) for x in "qkv")
    args = (None, c["type"], c["b"], c["m"], c["n"], c["d"], q, k, v)
    rest = (c["blocks"], c["count"], c["scale"], None, None, 0)
    assert abi.lib().tpu3_block_attn_fwd(*args, *rest, c["out"], None, c["rest"], None, 0) == want
    same = _heads(abi, heads=q.heads)
    # (the backward pass always needs a workspace)
    assert abi.lib().tpu3_block_attn_bwd(*args, same, same, *rest, 1 << 20, c["rest"], c["out"], 1 << 20, 1 << 20, None, 0) == want


def test_block_attention_backward_status(abi):
    h, f = _heads(abi), abi.lib().tpu3_block_attn_bwd
    need = abi.lib().tpu3_block_attn_bwd_workspace_bytes(1, 5, 40, 2, 2, 16, 4)
    def call(o=h, go=h, lse=1 << 20, dq=1 << 20, dk=1 << 20, dv=1 << 20, ws=1 << 20, size=need):
        return f(None, 0, 1, 5, 40, 16, h, h, h, o, go, 1 << 20, 4, 0.25, None, None, 0, lse, None, dq, dk, dv, ws, size)
    for change in (dict(o=_heads(abi, heads=1)), dict(go=_heads(abi, data=0)), dict(go=_heads(abi, sh=2)), dict(lse=None), dict(dq=0), dict(dq=8),
                   dict(dk=0), dict(dk=8), dict(dv=0), dict(dv=4), dict(ws=None), dict(ws=(1 << 20) + 8), dict(size=need - 1)):
        assert call(**change) == EINVAL


def test_tensors_that_are_not_on_a_gpu():
    ops = pkg("network.operations")
    x, k = torch.zeros((1, 4, 2, 16)), torch.zeros((1, 130, 1, 16))
    pos, freq = torch.zeros((1, 4)), ops.rotation_frequencies(1, 8)
    calls = [
        lambda: ops.norm_rotate(x, None, None, None, pos, freq), lambda: ops.block_means(k),
        lambda: ops.select_blocks(x, torch.zeros((1, 3, 1, 16)), 130, 2),
        lambda: ops.block_attention(x, k, k, torch.zeros((1, 4, 1, 2), dtype=torch.int32)),
        lambda: ops.sparse_attention(x, k, k, 2), lambda: ops.norm_rotate(None, None, None, None, pos, freq),
        lambda: ops.sparse_attention(x.numpy(), k, k, 2),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_frequencies():
    ops = pkg("network.operations")
    f = ops.rotation_frequencies(3, 4, base=100.0)
    assert f.dtype == torch.float64 and f.shape == (3, 4)
    assert torch.allclose(f[1], torch.tensor([1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert ops.rotation_frequencies(2, 0).shape == (2, 0)
