"""CPU tests of the dense operators' host side: what the C entry points refuse before anything is launched, tensors on the CPU, and
the 64-bit formulas that the GPU tests compare with."""
import ctypes as C

import pytest
import torch
import torch.nn.utils.parametrize

from dense_util import mlp_reference, norm_reference, normals
from mortar_amd import _lib, ops
from mortar_amd.block_sparse import CMSBlockLinear

A = 1 << 20                                   # an aligned address that is never read: every call here is refused


def _refused(rc, code=-1):
    assert rc == code and _lib.lib().mortar_last_error()


@pytest.mark.parametrize("fn", ["mortar_dense_linear", "mortar_dense_linear_dx", "mortar_dense_linear_dw"])
def test_dense_products(fn):
    f = getattr(_lib.lib(), fn)
    _refused(f(A, 8, 0, 64, A, 64, 64, 0, A, 64, None, None))                   # no columns
    _refused(f(A, -1, 64, 64, A, 64, 64, 0, A, 64, None, None))
    _refused(f(A, 8, 64, 64, A, 64, 64, 2, A, 64, None, None))                  # fp32
    _refused(f(None, 8, 64, 64, A, 64, 64, 0, A, 64, None, None))
    _refused(f(A, 8, 64, 64, None, 64, 64, 0, A, 64, None, None))
    _refused(f(A, 8, 64, 64, A, 64, 64, 0, None, 64, None, None))
    _refused(f(A + 2, 8, 64, 64, A, 64, 64, 0, A, 64, None, None))              # address
    _refused(f(A, 8, 64, 60, A, 64, 64, 0, A, 64, None, None))                  # leading dimension
    _refused(f(A, 8, 64, 56, A, 64, 64, 0, A, 64, None, None))
    _refused(f(A, 8, 64, 64, A, 64, 60, 0, A, 64, None, None))                  # width
    _refused(f(A, 8, 64, 1 << 23, A, 64, 64, 0, A, 64, None, None), -4)         # rows 16 MiB apart
    _refused(f(A, 8, 64, 64, A, 64, 64, 0, A, 1 << 23, None, None), -4)
    if fn != "mortar_dense_linear_dw":
        assert f(None, 0, 64, 64, None, 64, 64, 0, None, 64, None, None) == 0    # no rows: nothing to do
    else:
        _refused(f(A, 0, 64, 64, A, 64, 64, 0, A, 64, None, None))


def test_a_product_in_ranges_needs_its_workspace():
    L = _lib.lib()
    assert L.mortar_dense_workspace_bytes(100, 264, 9000) > 0
    _refused(L.mortar_dense_linear(A, 100, 9000, 9000, A, 9000, 264, 0, A, 264, None, None))
    assert L.mortar_dense_workspace_bytes(4096, 11264, 64) == 0 and L.mortar_dense_workspace_bytes(0, 8, 8) == 0


def test_swiglu_kernels():
    L = _lib.lib()
    up = lambda **k: L.mortar_dense_gateup_swiglu(*{**dict(x=A, M=8, d=64, ldx=64, w=A, ldw=64, f=64, t=0, h=A, ldh=64, gu=None, st=None), **k}.values())
    bwd = lambda **k: L.mortar_dense_swiglu_bwd(*{**dict(dy=A, M=8, d=64, ld=64, w=A, ldw=64, f=64, t=0, gu=A, dgu=A, ldg=128, h=None, ldh=64, st=None), **k}.values())
    for bad in (dict(M=-1), dict(d=0), dict(f=0), dict(t=2), dict(x=None), dict(w=None), dict(h=None), dict(ldx=60), dict(ldw=56), dict(ldh=56), dict(f=60), dict(gu=A + 8)):
        _refused(up(**bad))
    _refused(up(ldw=1 << 15, f=1 << 16))                                        # ldh < f
    _refused(up(ldw=1 << 15, f=1 << 16, ldh=1 << 16), -4)                       # gate and up rows 2 GiB and more apart
    for bad in (dict(M=-1), dict(d=0), dict(f=0), dict(t=2), dict(dy=None), dict(w=None), dict(gu=None), dict(dgu=None), dict(ldg=64), dict(h=A, ldh=56), dict(d=60)):
        _refused(bwd(**bad))
    assert up(M=0) == 0 and bwd(M=0) == 0


def test_layernorm():
    L = _lib.lib()
    fwd = lambda **k: L.mortar_layernorm(*{**dict(x=A, M=8, d=64, ldx=64, t=0, w=None, b=None, w32=0, eps=1e-5, y=A, ldy=64, mean=None, rstd=None, st=None), **k}.values())
    bwd = lambda **k: L.mortar_layernorm_bwd(*{**dict(dy=A, lddy=64, x=A, ldx=64, M=8, d=64, t=0, w=None, w32=0, mean=A, rstd=A, dx=A, lddx=64, dw=None, db=None, ws=None, st=None), **k}.values())
    for bad in (dict(M=-1), dict(d=0), dict(ldx=63), dict(ldy=63), dict(t=3), dict(x=None), dict(y=None), dict(mean=A)):
        _refused(fwd(**bad))
    for bad in (dict(M=0), dict(d=0), dict(ldx=63), dict(lddy=63), dict(lddx=63), dict(t=3), dict(x=None), dict(dy=None), dict(mean=None), dict(rstd=None), dict(dw=A)):
        _refused(bwd(**bad))
    assert fwd(M=0) == 0 and bwd(dx=None) == 0
    assert L.mortar_layernorm_workspace_bytes(10, 64) >= 2 * 64 * 4 and L.mortar_layernorm_workspace_bytes(0, 64) == 0


def test_fp8():
    L = _lib.lib()
    q = lambda **k: L.mortar_fp8_quantize(*{**dict(x=A, M=8, K=64, ldx=64, q=A, ldq=64, s=A, s_m=1, s_k=8, st=None), **k}.values())
    w = lambda **k: L.mortar_fp8_quantize_weight(*{**dict(w=A, N=8, K=64, ldw=64, t=0, q=A, ldq=64, s=A, s_n=1, st=None), **k}.values())
    y = lambda **k: L.mortar_fp8_linear(*{**dict(x=A, M=80, K=64, ldx=64, sx=A, s_m=1, s_k=80, w=A, ldw=64, sw=A, sw_n=1, N=64, y=A, ldy=64, ws=None, st=None), **k}.values())
    for bad in (dict(M=-1), dict(K=0), dict(K=72, ldx=72, ldq=80), dict(x=None), dict(q=None), dict(s=None), dict(ldx=60), dict(ldq=72), dict(x=A + 2), dict(q=A + 8)):
        _refused(q(**bad))
    _refused(q(K=128 * 65536, ldx=128 * 65536, ldq=128 * 65536), -4)
    for bad in (dict(N=0), dict(K=72, ldw=72, ldq=80), dict(t=5), dict(w=None), dict(q=None), dict(s=None), dict(s_n=0), dict(ldq=72)):
        _refused(w(**bad))
    for bad in (dict(M=-1), dict(K=72, ldx=80, ldw=80), dict(N=0), dict(N=60), dict(sw_n=0), dict(x=None), dict(w=None), dict(sw=None), dict(y=None), dict(ldx=72), dict(ldw=72),
                dict(ldy=60), dict(sx=None), dict(x=A + 8)):
        _refused(y(**bad))
    _refused(y(s_m=1 << 40), -4)
    _refused(y(N=1 << 26, ldy=1 << 26), -4)
    assert q(M=0) == 0 and y(M=0) == 0
    assert L.mortar_fp8_quantizes_inside(1, 2048) == 1 and L.mortar_fp8_quantizes_inside(17, 128) == 0 and L.mortar_fp8_quantizes_inside(16, 2048) == 0


def test_tensors_on_the_cpu_are_refused():
    x, w = torch.zeros(4, 32), torch.zeros(64, 32)
    for call in (lambda: ops.layernorm(x), lambda: ops.dense_mlp(x, w, w.t()), lambda: ops.quantize_fp8(x), lambda: ops.quantize_fp8_weight(w), lambda: ops.linear_fp8(x, w, w)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()
    for call in (lambda: ops.layernorm(None), lambda: ops.dense_mlp(x.numpy(), w, w), lambda: ops.layernorm(torch.zeros(4, device="meta"))):
        with pytest.raises((TypeError, RuntimeError)):
            call()


def test_formulas_against_autograd_and_differences():
    """The references in 64 bits: torch's own gradients of the same forward, and central differences."""
    x, w, b, dy = (normals(s, i, torch.float64, "cpu").requires_grad_(True) for i, s in enumerate(((6, 20), (20,), (20,), (6, 20))))
    y, *grads = norm_reference(x, w, b, 1e-3, dy)
    ref = torch.nn.functional.layer_norm(x, (20,), w, b, 1e-3)
    assert torch.allclose(y, ref, rtol=1e-12, atol=1e-12)
    for g, r in zip(grads, torch.autograd.grad(ref, (x, w, b), dy)):
        assert torch.allclose(g, r, rtol=1e-10, atol=1e-10)
    x, g, d, dy = (normals(s, 9 + i, torch.float64, "cpu") for i, s in enumerate(((5, 16), (48, 16), (16, 24), (5, 16))))
    _, *grads = mlp_reference(x, g, d, dy)
    for i, grad in enumerate(grads):
        v, e = normals(grad.shape, 50 + i, torch.float64, "cpu"), 1e-4
        at = lambda s: float((dy * mlp_reference(*[p + s * v if j == i else p for j, p in enumerate((x, g, d))])).sum())
        assert abs((at(e) - at(-e)) / (2 * e) - float((grad * v).sum())) <= 1e-5 * float(grad.abs().sum())


def test_a_parametrised_weight_is_the_layers_weight():
    """The uncarved layer reads its weight as an attribute: under a parametrisation it is no parameter of the module."""
    lin = CMSBlockLinear(32, 48)
    w, x = lin.weight.detach().clone(), normals((3, 32), 1, torch.float32, "cpu")
    torch.nn.utils.parametrize.register_parametrization(lin, "weight", Doubled())
    assert "weight" not in lin._parameters
    assert torch.equal(lin(x), torch.nn.functional.linear(x, 2 * w, lin.bias))
    assert torch.equal(lin.dense_weight(), 2 * w)


class Doubled(torch.nn.Module):
    def forward(self, w):
        return 2 * w


def test_layers_that_cannot_be_packed():
    """Widths that the 8-bit product does not take are refused before the layer is touched, carved and packed layers likewise."""
    from mortar_amd.deploy_quant import pack_dense_fp8
    for shape in ((20, 32), (32, 12)):
        lin = CMSBlockLinear(*shape, tile_size=4)
        with pytest.raises(ValueError, match="not a multiple"):
            pack_dense_fp8(lin)
        assert "weight" in lin._parameters
    lin = CMSBlockLinear(32, 32)
    lin.carve()
    with pytest.raises(AssertionError):
        pack_dense_fp8(lin)
    lin = CMSBlockLinear(32, 32)
    with pytest.raises(RuntimeError, match="ROCm device"):
        pack_dense_fp8(lin)
    assert "weight" in lin._parameters and not lin._buffers.keys() & {"dense_fp8"}
