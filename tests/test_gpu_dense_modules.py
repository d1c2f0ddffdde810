"""The modules that run the dense operators: the uncarved MLP with dense_fused, a training step of norm and MLP together, layers packed to 8 bits."""
import copy
import io

import pytest
import torch
import torch.nn.functional as F

import mortar_amd
from dense_util import assert_within, fp8_reference, fp8_rows, fp8_weight, mlp_bounds, mlp_reference, norm_bounds, norm_reference, normals
from mortar_amd import deploy_quant, ops
from mortar_amd.block_sparse import CMSBlockLinear
from mortar_amd.mlp import _SwiGLUMortar

pytestmark = pytest.mark.gpu


def _mlp(dev, t=torch.bfloat16, d=64, f=96, seed=0):
    torch.manual_seed(seed)
    return _SwiGLUMortar(d, f).to(dev).to(t)


@pytest.mark.parametrize("M", [3, 70])
def test_uncarved_module_fused(dev, M):
    mlp = _mlp(dev)
    x, dy = normals((2, M, 64), 1, torch.bfloat16, dev).requires_grad_(True), normals((2, M, 64), 2, torch.bfloat16, dev)
    params = [mlp.gate_up._cms.weight, mlp.down._cms.weight]
    args = (x.detach().reshape(-1, 64), *[p.detach() for p in params])
    plain = mlp(x)
    mlp.dense_fused = True
    y = mlp(x)
    got = (y, *torch.autograd.grad(y, [x, *params], dy))
    assert y.shape == plain.shape
    for g, r, e in zip(got, mlp_reference(*args, dy.reshape(-1, 64)), mlp_bounds(*args, dy.reshape(-1, 64))):
        assert_within(g.detach().reshape(r.shape), r, e, "fused")
    with torch.no_grad():
        assert torch.equal(mlp(x), ops.dense_mlp(x, *params))
    mlp.dense_fused = False
    assert torch.equal(mlp(x), plain)


def test_pruned_tiles_stay_zero_and_get_no_gradient(dev):
    mlp = _mlp(dev)
    mlp.dense_fused = True
    cms = mlp.gate_up._cms
    mask = torch.rand(cms.R, cms.C, generator=torch.Generator().manual_seed(1)) > 0.5
    cms.set_block_mask(mask.to(dev))
    x = normals((9, 64), 1, torch.bfloat16, dev)
    full = mask.to(dev).repeat_interleave(16, 0).repeat_interleave(16, 1)
    y = mlp(x)
    assert torch.equal(y, ops.dense_mlp(x, cms.weight * full, mlp.down._cms.weight))
    (g,) = torch.autograd.grad(y.sum(), [cms.weight])
    assert not g[~full].any() and bool(g[full].any())


def test_calls_that_the_fused_form_leaves_alone(dev, monkeypatch):
    """fp32 layers, mixed types, hooks, subclasses, autocast, a router: torch's layers run, with their results."""
    monkeypatch.setattr(ops, "dense_mlp", lambda *a: pytest.fail("fused"))
    x = normals((5, 64), 1, torch.float32, dev)
    for change in ("fp32", "hook", "autocast", "router", "override"):
        mlp = _mlp(dev, torch.float32 if change in ("fp32", "autocast", "router") else torch.bfloat16)
        mlp.dense_fused = True
        xx = x if change in ("fp32", "autocast", "router") else x.bfloat16()
        seen = []
        if change == "hook":
            mlp.down.register_forward_hook(lambda *a: seen.append(1))
        if change == "override":
            mlp.gate_up._cms.forward = lambda v: seen.append(1) or CMSBlockLinear.forward(mlp.gate_up._cms, v)
        if change == "router":
            mlp.enable_routing(n_clusters=4)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=change == "autocast"):
            y = mlp(xx)
        assert y.shape == (5, 64) and (seen == [1]) == (change in ("hook", "override"))


def test_norm_and_mlp_in_one_training_step(dev):
    """A block as it is trained before the carve: LayerNorm, MLP, residual; each part within its own bound on the other's outputs."""
    t = torch.bfloat16
    mlp = _mlp(dev)
    mlp.dense_fused = True
    x, dy = normals((40, 64), 3, t, dev).requires_grad_(True), normals((40, 64), 4, t, dev)
    nw, nb = (1 + normals((64,), 5, torch.float32, dev, 0.1)).requires_grad_(True), normals((64,), 6, torch.float32, dev, 0.1).requires_grad_(True)
    wg, wd = mlp.gate_up._cms.weight, mlp.down._cms.weight
    z = ops.layernorm(x, nw, nb)
    z.retain_grad()
    out = x + mlp(z)
    out.backward(dy)
    assert_within(z.detach(), norm_reference(x.detach(), nw.detach(), nb.detach(), 1e-5), norm_bounds(x.detach(), nw.detach(), nb.detach(), 1e-5), "norm")
    args = (z.detach(), wg.detach(), wd.detach(), dy)
    for g, r, e in zip((z.grad, wg.grad, wd.grad), mlp_reference(*args)[1:], mlp_bounds(*args)[1:]):
        assert_within(g, r, e, "mlp")
    _, dx, dw, db = norm_reference(x.detach(), nw.detach(), nb.detach(), 1e-5, z.grad)
    _, ex, ew, eb = norm_bounds(x.detach(), nw.detach(), nb.detach(), 1e-5, z.grad)
    assert_within(x.grad, dx + dy.double(), 2 * ex + 2.0 ** -8 * (dx + dy.double()).abs(), "dx")           # the sum with the residual's is rounded once more
    assert_within(nw.grad, dw, ew + 2.0 ** -24 * dw.abs(), "dw")
    assert_within(nb.grad, db, eb + 2.0 ** -24 * db.abs(), "db")


def test_layer_packed_to_8_bits(dev):
    torch.manual_seed(3)
    lin = mortar_amd.MortarLinear(160, 272, bias=True).to(dev)
    torch.nn.init.normal_(lin.bias)
    w = lin._cms.weight.detach().clone()
    info = deploy_quant.pack_dense_fp8(lin._cms)
    assert "weight" not in lin._cms._parameters and info["relative_error"] <= 2.0 ** -4 and info["packed_bytes"] == 272 * 160 + 4 * 3 * 2
    q, s = fp8_weight(w)
    for x in (normals((3, 160), 1, torch.bfloat16, dev), normals((2, 50, 160), 2, torch.bfloat16, dev), normals((3, 160), 1, torch.float32, dev)):
        y = lin(x)
        x2 = x.reshape(-1, 160).bfloat16()
        xq, xs = fp8_rows(x2.cpu())
        ref, bound = fp8_reference(xq.to(dev), xs.to(dev), q, s)
        b = lin.bias.detach().double()
        assert y.shape == (*x.shape[:-1], 272)
        assert y.dtype == x.dtype                          # the sum with the bias, in fp32, is rounded to the activations' type
        assert_within(y.detach().reshape(-1, 272), ref + b, bound + 2.0 ** -8 * (bound + (ref + b).abs()) + 2.0 ** -24 * (ref + b).abs(), "y")
    with pytest.raises(RuntimeError, match="inference only"):
        lin(normals((3, 160), 1, torch.bfloat16, dev).requires_grad_(True))
    with pytest.raises(AssertionError):
        deploy_quant.pack_dense_fp8(lin._cms)
    with pytest.raises(AssertionError):
        lin.carve()


def test_packed_layers_save_load_copy_and_cast(dev):
    mlp = _mlp(dev, torch.float32)
    for m in (mlp.gate_up, mlp.down):
        deploy_quant.pack_dense_fp8(m._cms)
    x = normals((7, 64), 1, torch.bfloat16, dev)
    y = mlp(x)
    buf = io.BytesIO()
    torch.save(mlp.state_dict(), buf)
    buf.seek(0)
    other = _SwiGLUMortar(64, 96).to(dev)
    other.load_state_dict(torch.load(buf, weights_only=True))
    assert torch.equal(other(x), y) and torch.equal(copy.deepcopy(mlp)(x), y)
    h = F.silu(mlp.gate_up(x).chunk(2, -1)[0]) * mlp.gate_up(x).chunk(2, -1)[1]
    assert torch.equal(mlp.down(h), y)
    cast = copy.deepcopy(mlp).bfloat16()
    assert torch.equal(cast.gate_up._cms.dense_fp8, mlp.gate_up._cms.dense_fp8)
    with pytest.raises(TypeError):                       # scales in 16 bits are refused, not used
        cast(x)


def test_pruned_layer_packed(dev):
    torch.manual_seed(5)
    lin = mortar_amd.MortarLinear(64, 64, bias=False).to(dev)
    mask = torch.eye(4, dtype=torch.bool)
    lin._cms.set_block_mask(mask.to(dev))
    deploy_quant.pack_dense_fp8(lin._cms)
    full = mask.repeat_interleave(16, 0).repeat_interleave(16, 1).to(dev)
    assert not lin._cms.dense_fp8.view(torch.float8_e4m3fn).float()[~full].any()             # a pruned negative weight is -0: code 128
