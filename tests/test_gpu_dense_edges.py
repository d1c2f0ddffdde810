"""Calls at the edges of the dense operators: what hangs on the layers of a fused MLP, calls that only torch's layers cover, rows far apart, values
at the ends of the range, gradients and scales in unusual forms."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from dense_util import assert_within, normals, rounding
from mortar_amd import _lib, ops
from mortar_amd.mlp import _SwiGLUMortar

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _mlp(dev, d=64, f=96, t=BF16):
    torch.manual_seed(0)
    mlp = _SwiGLUMortar(d, f).to(dev).to(t)
    mlp.dense_fused = True
    return mlp


# ---- the MLP's modules


@pytest.mark.parametrize("kind", ["backward", "backward_pre", "global_backward", "global_backward_pre"])
@pytest.mark.parametrize("where", ["gate_up", "gate_up._cms", "down", "down._cms"])
def test_backward_hooks_of_the_layers_run(dev, where, kind):
    mlp = _mlp(dev)
    m, seen = mlp.get_submodule(where), []
    see = lambda mod, *a: seen.append(mod) if mod is m else None
    if kind == "backward":
        handle = m.register_full_backward_hook(see)
    elif kind == "backward_pre":
        handle = m.register_full_backward_pre_hook(see)
    elif kind == "global_backward":
        handle = torch.nn.modules.module.register_module_full_backward_hook(see)
    else:
        handle = torch.nn.modules.module.register_module_full_backward_pre_hook(see)
    try:
        x = normals((5, 64), 1, BF16, dev).requires_grad_(True)
        mlp(x).sum().backward()
    finally:
        handle.remove()
    assert seen == [m]


def _apart(t, pitch):
    """The rows of t `pitch` values apart."""
    bits = torch.uint8 if t.element_size() == 1 else torch.int16
    wide = torch.zeros((t.shape[0], pitch), dtype=bits, device=t.device)
    wide[:, -t.shape[1]:] = t.view(bits)
    return wide.view(t.dtype)[:, -t.shape[1]:]


# ---- rows far apart


def test_mlp_of_rows_far_apart(dev):
    """Rows 2^22 values and more apart, as the last token of every sequence of hidden states has them; the same bits as those of the copy."""
    hidden = torch.zeros((2, 2048, 2048), dtype=BF16, device=dev)
    hidden[:, -1] = normals((2, 2048), 1, BF16, dev)
    wgu, wd = normals((48, 2048), 2, BF16, dev, 0.02), normals((2048, 24), 3, BF16, dev, 0.2)
    want = ops.dense_mlp(hidden[:, -1].contiguous(), wgu, wd)
    assert torch.equal(ops.dense_mlp(hidden[:, -1], wgu, wd), want) and torch.equal(ops.dense_mlp(hidden[:, -1:], wgu, wd), want[:, None])
    few = hidden[:, -1].repeat(5, 1)
    assert torch.equal(ops.dense_mlp(_apart(few, 1 << 22), wgu, wd), ops.dense_mlp(few, wgu, wd))
    wd = wd[:64]
    assert torch.equal(ops.dense_mlp(few, _apart(wgu, 1 << 22), _apart(wd, 1 << 22)), ops.dense_mlp(few, wgu, wd))


def test_gradient_of_rows_far_apart(dev):
    x, wgu, wd = normals((2, 64), 1, BF16, dev), normals((48, 64), 2, BF16, dev, 0.1), normals((2048, 24), 3, BF16, dev, 0.2)
    dy = torch.zeros((2, 2048, 2048), dtype=BF16, device=dev)
    dy[:, 5] = normals((2, 2048), 4, BF16, dev)
    leaves = [v.requires_grad_(True) for v in (x, wgu, wd)]
    want = torch.autograd.grad(ops.dense_mlp(*leaves), leaves, dy[:, 5].contiguous())
    got = torch.autograd.grad(ops.dense_mlp(*leaves), leaves, dy[:, 5])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M", [2, 20, 70])
def test_codes_of_rows_far_apart(dev, M):
    x = normals((M, 160), 1, BF16, dev)
    wq, ws = ops.quantize_fp8_weight(normals((72, 160), 2, torch.float32, dev, 0.1))
    q, s = ops.quantize_fp8(x)
    want = ops.linear_fp8(q, wq, ws, s)
    assert torch.equal(ops.linear_fp8(_apart(q, 1 << 23), wq, ws, s), want)
    far = _apart(x, 1 << 22)
    assert torch.equal(ops.linear_fp8(far, wq, ws), want) and torch.equal(ops.quantize_fp8(far)[0].view(torch.uint8), q.view(torch.uint8))
