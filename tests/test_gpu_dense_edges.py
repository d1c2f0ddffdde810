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


class _Sub(torch.Tensor):
    seen = 0

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        if func is torch.nn.functional.linear:
            cls.seen += 1
        return super().__torch_function__(func, types, args, kwargs or {})


class _Watch(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


def test_calls_that_only_torchs_layers_cover(dev):
    """Functional transforms, tracing, forward mode, subclasses, modes: the results of the layers, not an exception."""
    mlp = _mlp(dev)
    x, t = normals((3, 64), 1, BF16, dev), normals((3, 64), 2, BF16, dev)
    plain = _mlp(dev)
    plain.dense_fused = False

    def equal(f):
        a, b = f(mlp), f(plain)
        assert all(torch.equal(p, q) for p, q in zip(a, b)) if isinstance(a, tuple) else torch.equal(a, b)
    equal(lambda m: torch.func.vmap(m)(x.view(3, 1, 64)))
    equal(lambda m: torch.func.jvp(m, (x,), (t,)))
    equal(lambda m: torch.func.grad(lambda v: m(v).float().sum())(x))
    equal(lambda m: torch.jit.trace(m, x, check_trace=False)(x))
    equal(lambda m: torch.compile(m, backend="eager", fullgraph=True)(x))

    def forward_mode(m):
        with torch.autograd.forward_ad.dual_level():
            y = torch.autograd.forward_ad.unpack_dual(m(torch.autograd.forward_ad.make_dual(x, t)))
            return y.primal, y.tangent
    equal(forward_mode)

    def weights_tangent(m):
        w = m.down._cms.weight
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(w.detach(), torch.ones_like(w))
            y = torch.autograd.forward_ad.unpack_dual(torch.func.functional_call(m, {"down._cms.weight": dual}, (x,)))
            return y.primal, y.tangent
    equal(weights_tangent)
    with _Watch() as watch:
        y = mlp(x)
    assert torch.equal(y, plain(x)) and sum("mm" in n or "linear" in n for n in watch.names) == 2
    y = mlp(x.as_subclass(_Sub))
    assert type(y) is _Sub and _Sub.seen == 2 and torch.equal(y.as_subclass(torch.Tensor), plain(x))


def test_the_second_derivative_is_refused(dev):
    x = normals((3, 64), 1, BF16, dev).requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(_mlp(dev)(x).sum(), [x], create_graph=True)


def test_weights_that_one_launch_cannot_address(dev):
    """gate_up of 2 GiB for the gate rows alone (one value, repeated): torch's layers run."""
    n = 1 << 15
    mlp = _mlp(dev)
    one = lambda *s: torch.nn.Parameter(torch.full((), 2.0 ** -15, dtype=BF16, device=dev).expand(s), requires_grad=False)
    mlp.gate_up._cms.weight, mlp.down._cms.weight = one(2 * n, n), one(n, n)
    y = mlp(torch.ones((1, n), dtype=BF16, device=dev))
    h = torch.nn.functional.silu(torch.ones((), dtype=BF16, device=dev))           # gate = up = 1 exactly, y the mean of n values of h
    assert torch.equal(y, h.expand(1, n))


@pytest.mark.parametrize("M", [3, 70])
def test_gate_and_up_rows_far_apart(dev, M):
    """A gate row and its up row 2 GiB apart, in rows that are not."""
    x, wgu, wd = normals((M, 64), 1, BF16, dev), normals((2048, 64), 2, BF16, dev, 0.1), normals((16, 1024), 3, BF16, dev, 0.03)
    assert torch.equal(ops.dense_mlp(x, _apart(wgu, 1 << 20), wd), ops.dense_mlp(x, wgu, wd))


def test_scales_of_other_rows_are_refused(dev):
    wq, ws = ops.quantize_fp8_weight(normals((72, 160), 1, torch.float32, dev, 0.1))
    q, s = ops.quantize_fp8(normals((2, 3, 160), 2, BF16, dev))
    assert ops.linear_fp8(q, wq, ws, s).shape == (2, 3, 72)
    for other in (s.transpose(0, 1), s.reshape(3, 2, 2), s.reshape(6, 1, 2)):
        with pytest.raises(ValueError, match="x_scale must be"):
            ops.linear_fp8(q, wq, ws, other)


def test_scales_of_a_weight_that_are_repeated(dev):
    wq, ws = ops.quantize_fp8_weight(normals((264, 272), 1, torch.float32, dev, 0.1))
    x = normals((4, 272), 2, BF16, dev)
    for rows in (x, x.repeat(20, 1)):
        for view in (ws[:1].expand(3, 3), ws[:, :1].expand(3, 3), ws[0, 0].expand(3, 3)):
            assert torch.equal(ops.linear_fp8(rows, wq, view), ops.linear_fp8(rows, wq, view.clone()))


# ---- gradients and scales in unusual forms


def test_gradients_that_are_negated_lazily(dev):
    """A gradient with the negative bit, as the imaginary part of a conjugate has it."""
    x, w, b = normals((6, 64), 1, BF16, dev).requires_grad_(True), normals((64,), 2, BF16, dev).requires_grad_(True), normals((64,), 3, BF16, dev).requires_grad_(True)
    wgu, wd, dy = normals((48, 64), 4, BF16, dev, 0.1).requires_grad_(True), normals((64, 24), 5, BF16, dev, 0.2).requires_grad_(True), normals((6, 64), 6, BF16, dev)
    for leaves, f in (((x, w, b), ops.layernorm), ((x, wgu, wd), ops.dense_mlp)):
        want = torch.autograd.grad(f(*leaves), leaves, -dy)
        got = torch.autograd.grad(f(*leaves), leaves, torch._neg_view(dy))
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_batched_gradients_are_refused(dev):
    x, w = normals((6, 64), 1, BF16, dev).requires_grad_(True), normals((64,), 2, BF16, dev)
    wgu, wd, dy = normals((48, 64), 4, BF16, dev, 0.1), normals((64, 24), 5, BF16, dev, 0.2), normals((2, 6, 64), 6, BF16, dev)
    for y in (ops.layernorm(x, w), ops.dense_mlp(x, wgu, wd)):
        with pytest.raises(RuntimeError, match="plain strided tensor"):
            torch.autograd.grad(y, [x], dy, is_grads_batched=True)


def test_a_mode_that_watches_the_backward(dev):
    """Forward calls inside a dispatch mode are left to torch; a backward inside one has plain gradients and runs."""
    x = normals((6, 64), 1, BF16, dev).requires_grad_(True)
    wgu, wd, dy = normals((48, 64), 4, BF16, dev, 0.1), normals((64, 24), 5, BF16, dev, 0.2), normals((6, 64), 6, BF16, dev)
    for f in (lambda: ops.layernorm(x), lambda: ops.dense_mlp(x, wgu, wd)):
        (want,) = torch.autograd.grad(f(), [x], dy)
        y = f()
        with _Watch():
            (got,) = torch.autograd.grad(y, [x], dy)
        assert torch.equal(got, want)


# ---- values at the ends of the range


@pytest.mark.parametrize("t", [torch.float32, BF16], ids=str)
@pytest.mark.parametrize("d", [16, 40, 1000, 1544, 5000])
@pytest.mark.parametrize("params", [True, False])
def test_rows_around_a_large_mean_have_a_gradient(dev, params, d, t):
    """x = mean = 2^120 and 1 / deviation = 2^9: what lies beyond the row in registers, (0 - mean) / deviation there, is not finite.
    z = 0, so dx = r (g - mean(g)), dw = 0 and db = sum of dy; d fills neither a vector's, a wave's nor a workgroup's last lanes."""
    M, r = 5, 2.0 ** 9
    w, dy = normals((d,), 1, torch.float32, dev).to(t), normals((M, d), 2, torch.float32, dev).to(t)
    mean, rstd = torch.full((M,), 2.0 ** 120, device=dev), torch.full((M,), r, device=dev)
    L = _lib.lib()
    ws = torch.full((L.mortar_layernorm_workspace_bytes(M, d) // 4,), float("nan"), device=dev)
    for off in (0, 1):
        x = torch.full((M, d + off), 2.0 ** 120, dtype=t, device=dev)[:, off:]
        dx, dw, db = torch.full((M, d), float("nan"), dtype=t, device=dev), torch.full((d,), float("nan"), dtype=t, device=dev), torch.full((d,), float("nan"), dtype=t, device=dev)
        ptr = lambda v: v.data_ptr() if params else None
        _lib.check(L.mortar_layernorm_bwd(dy.data_ptr(), d, x.data_ptr(), x.stride(0), M, d, {torch.float32: 2, BF16: 0}[t], w.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(),
                                          dx.data_ptr(), d, ptr(dw), ptr(db), ptr(ws), torch.cuda.current_stream().cuda_stream), "layernorm_bwd")
        g = dy.double() * w.double()
        ref = r * (g - g.mean(1, keepdim=True))
        chain = 2.0 ** -24 * (72 + d // 256 + 10)                   # as dense_util.norm_bounds: the products, their sum, the difference
        assert_within(dx, ref, 2 * r * (2.0 ** -23 * g.abs() + chain * g.abs().mean(1, keepdim=True)) + rounding(t, ref), "dx")
        if params:
            assert not dw.any()
            ref = dy.double().sum(0)
            assert_within(db, ref, 2.0 ** -24 * M * dy.double().abs().sum(0) + rounding(t, ref), "db")


@pytest.mark.parametrize("exponent", [-149, -147, -145, -142, -141, -140, -139, -138, -137, -136, -135, -130, -120])
def test_weights_of_hardly_any_size(dev, exponent):
    """Blocks whose scale fp32 can hold only in a few bits or not at all: finite codes, the block's values or zeros, and finite results."""
    w = torch.zeros((136, 272))
    w[:128, :128] = normals((128, 128), 1, torch.float32, "cpu", 0.1)
    w[:128, 128:256] = (torch.linspace(1.0, 1.99, 128).double() * 2.0 ** exponent).float()
    w[128:, :128] = 2.0 ** exponent
    q, s = ops.quantize_fp8_weight(w.to(dev))
    codes, sizes = q.cpu().float().double(), s.cpu().double()
    v = codes * sizes.repeat_interleave(128, 0)[:136].repeat_interleave(128, 1)[:, :272]
    assert not v.isnan().any() and bool((sizes > 0).all())
    for block in ((slice(0, 128), slice(128, 256)), (slice(128, 136), slice(0, 128))):
        a, r, sc = w[block].double(), v[block], float(sizes[block[0].start // 128, block[1].start // 128])
        if exponent <= -138:                             # amax / 448 below 2^-145: nothing that 8 bits could hold beside a scale
            assert sc == 1.0 and not r.any()
        elif exponent >= -135:                           # a step of e4m3 at most from it: half of 2^-3, and the scale's own rounding, 1/32 at most, at the top
            assert sc < 1e-30 and bool(((r - a).abs() <= a.abs() * 2.0 ** -3).all())
    x = normals((5, 272), 2, BF16, dev)
    for rows in (x, x.repeat(20, 1)):
        y = ops.linear_fp8(rows, q, s)
        assert bool(y.isfinite().all())


def test_few_rows_take_no_scratch(dev):
    """Up to 8 rows a forward call allocates its result and the hidden activations, and nothing else."""
    wgu, wd = normals((11264, 256), 1, BF16, dev, 0.06), normals((264, 5632), 2, BF16, dev, 0.02)
    for M in (1, 8):
        x = normals((M, 256), 3, BF16, dev)
        ops.dense_mlp(x, wgu, wd)
        count = lambda: torch.cuda.memory_stats()["allocation.all.allocated"]
        before = count()
        y = ops.dense_mlp(x, wgu, wd)
        assert count() - before == 2 and y.shape == (M, 264)


def test_saved_tensors_that_come_back_in_other_strides(dev):
    """Saved-tensor hooks hand back the same values: elsewhere, transposed, or by way of the host."""
    x, w, b = normals((6, 64), 1, BF16, dev).requires_grad_(True), normals((64,), 2, BF16, dev).requires_grad_(True), normals((64,), 3, BF16, dev).requires_grad_(True)
    wgu, wd, dy = normals((48, 64), 4, BF16, dev, 0.1).requires_grad_(True), normals((64, 24), 5, BF16, dev, 0.2).requires_grad_(True), normals((6, 64), 6, BF16, dev)
    turned = (lambda t: t.detach().t().contiguous(), lambda t: t.t())
    spread = (lambda t: t.detach().repeat_interleave(2, 0), lambda t: t[::2])
    host = (lambda t: t.detach().cpu(), lambda t: t.to(dev))
    for leaves, f in (((x, w, b), ops.layernorm), ((x, wgu, wd), ops.dense_mlp)):
        want = torch.autograd.grad(f(*leaves), leaves, dy)
        for pack, unpack in (turned, spread, host):
            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                y = f(*leaves)
            assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy), want))


@pytest.mark.parametrize("unpack", [lambda t: t.cpu(), lambda t: t[:1], lambda t: t.float() if t.is_floating_point() else t.int(), lambda t: t.unsqueeze(0)], ids=["host", "shape", "type", "dims"])
def test_saved_tensors_that_come_back_as_others_are_refused(dev, unpack):
    x, w = normals((6, 64), 1, BF16, dev).requires_grad_(True), normals((64,), 2, BF16, dev)
    wgu, wd, dy = normals((48, 64), 4, BF16, dev, 0.1), normals((64, 24), 5, BF16, dev, 0.2), normals((6, 64), 6, BF16, dev)
    for f in (lambda: ops.layernorm(x, w), lambda: ops.dense_mlp(x, wgu, wd)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
            y = f()
        with pytest.raises(RuntimeError, match="came back"):
            torch.autograd.grad(y, [x], dy)


@pytest.mark.parametrize("M", [1, 20, 70])
def test_scales_of_rows_far_apart(dev, M):
    """x_scale whose rows span 2 GiB, in one matrix or as the last of every sequence's."""
    wq, ws = ops.quantize_fp8_weight(normals((72, 160), 1, torch.float32, dev, 0.1))
    q, s = ops.quantize_fp8(normals((M, 160), 2, BF16, dev))
    wide = torch.zeros((M, (1 << 29) // M + 8), device=dev)
    wide[:, -2:] = s
    want = ops.linear_fp8(q, wq, ws, s)
    assert torch.equal(ops.linear_fp8(q, wq, ws, wide[:, -2:]), want)
    assert torch.equal(ops.linear_fp8(q[:, None], wq, ws, wide[:, None, -2:]), want[:, None])
