"""Dense operators on tensors whose byte offsets pass 32 bits: the last rows against the 64-bit formulas of those rows alone."""
import pytest
import torch

from dense_util import assert_within, fp8_reference, mlp_bounds, mlp_reference, norm_bounds, norm_reference, normals
from mortar_amd import ops

pytestmark = pytest.mark.gpu
TAIL = 40


def _rows(M, d, dev, seed):
    """M rows of which the last are random (the others: one random row)."""
    x = normals((1, d), seed, torch.bfloat16, dev).expand(M, d).contiguous()
    x[-TAIL:] = normals((TAIL, d), seed + 1, torch.bfloat16, dev)
    return x


def test_layernorm(dev):
    x = _rows((1 << 21) + 3, 1040, dev, 1)
    assert x.numel() * 2 > 1 << 32
    w, b = normals((1040,), 3, torch.bfloat16, dev), normals((1040,), 4, torch.bfloat16, dev)
    dy = torch.zeros_like(x)
    dy[-TAIL:] = normals((TAIL, 1040), 5, torch.bfloat16, dev)
    leaf = x.requires_grad_(True)
    y = ops.layernorm(leaf, w, b)
    (dx,) = torch.autograd.grad(y, [leaf], dy)
    args = (x.detach()[-TAIL:], w, b, 1e-5)
    assert_within(y.detach()[-TAIL:], norm_reference(*args), norm_bounds(*args), "y")
    assert_within(dx[-TAIL:], norm_reference(*args, dy[-TAIL:])[1], norm_bounds(*args, dy[-TAIL:])[1], "dx")
    assert not dx[:-TAIL].any()


def test_mlp_rows(dev):
    x = _rows((1 << 21) + 3, 1040, dev, 1)
    wgu, wd = normals((16, 1040), 6, torch.bfloat16, dev, 0.03), normals((8, 8), 7, torch.bfloat16, dev)
    y = ops.dense_mlp(x, wgu, wd)
    args = (x[-TAIL:], wgu, wd)
    assert_within(y[-TAIL:], mlp_reference(*args), mlp_bounds(*args), "y")
    assert torch.equal(y[:-TAIL], y[:1].expand(y.shape[0] - TAIL, -1))


def test_mlp_kept_values(dev):
    """The gate_up output in 24 bits is the largest tensor here (4.9 GB)."""
    M, f = 400003, 2048
    assert 6 * M * f > 1 << 32
    x = _rows(M, 64, dev, 1).requires_grad_(True)
    wgu, wd = normals((2 * f, 64), 6, torch.bfloat16, dev, 0.1), normals((16, f), 7, torch.bfloat16, dev, 0.03)
    dy = torch.zeros((M, 16), dtype=torch.bfloat16, device=dev)
    dy[-TAIL:] = normals((TAIL, 16), 8, torch.bfloat16, dev)
    wgu.requires_grad_(True), wd.requires_grad_(True)
    y = ops.dense_mlp(x, wgu, wd)
    dx, dgu, dwd = torch.autograd.grad(y, [x, wgu, wd], dy)
    args = (x.detach()[-TAIL:], wgu.detach(), wd.detach(), dy[-TAIL:])          # the other rows' gradients are zero, their sums too
    for g, r, e in zip((y.detach()[-TAIL:], dx[-TAIL:], dgu, dwd), mlp_reference(*args), mlp_bounds(*args)):
        assert_within(g, r, e, "mlp")
    assert not dx[:-TAIL].any()


def test_fp8(dev):
    x = _rows((1 << 22) + 3, 1040, dev, 1)
    wq, ws = ops.quantize_fp8_weight(normals((8, 1040), 6, torch.bfloat16, dev, 0.03))
    q, s = ops.quantize_fp8(x)
    assert q.numel() > 1 << 32
    tq, ts = ops.quantize_fp8(x[-TAIL:])
    assert torch.equal(q[-TAIL:].view(torch.uint8), tq.view(torch.uint8)) and torch.equal(s[-TAIL:], ts)
    ref, bound = fp8_reference(tq, ts, wq, ws)
    for y in (ops.linear_fp8(x, wq, ws), ops.linear_fp8(q, wq, ws, s)):
        assert_within(y[-TAIL:], ref, bound, "y")
        assert torch.equal(y[:-TAIL], y[:1].expand(y.shape[0] - TAIL, -1))
