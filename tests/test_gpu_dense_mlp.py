"""The dense products and ops.dense_mlp.  Products of integers are exact in fp32, so every tile, tail and split has to give the rounded
integer; the whole MLP and its gradients are held to the bounds of dense_util.mlp_bounds."""
import pytest
import torch

from dense_util import assert_within, ints, mlp_bounds, mlp_reference, normals, rounding
from mortar_amd import _lib, ops

pytestmark = pytest.mark.gpu
TYPES = {torch.bfloat16: 0, torch.float16: 1}


def _padded(rows, cols, extra, t, dev, fill=float("nan")):
    """A [rows, cols] matrix inside a wider and longer one filled with NaN."""
    whole = torch.full((rows + 3, cols + extra), fill, dtype=t, device=dev)
    return whole, whole[:rows, :cols]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ws(n, dev):
    return torch.full((max(n, 16) // 4,), float("nan"), dtype=torch.float32, device=dev)


def _product(form, M, N, K, t, dev, seed, extra=0):
    """One of the three products through the C-ABI on integers, operands and result inside matrices of NaN; -> (result, exact, surroundings intact)."""
    L = _lib.lib()
    most = 3
    p_shape, q_shape = {"y": ((N, K), (M, K)), "dx": ((K, N), (M, K)), "dw": ((K, N), (K, M))}[form]
    P, Q = ints(p_shape, most, seed, t, dev), ints(q_shape, most, seed + 1, t, dev)
    pw, p = _padded(*p_shape, extra, t, dev)
    qw, q = _padded(*q_shape, extra, t, dev)
    cw, c = _padded(M, N, extra, t, dev)
    p.copy_(P), q.copy_(Q)
    n = L.mortar_dense_workspace_bytes(M, N, K)
    ws = _ws(n, dev)
    head = (q.data_ptr(), K if form == "dw" else M, M if form == "dw" else K, q.stride(0), p.data_ptr(), p.stride(0), N)
    fn = {"y": L.mortar_dense_linear, "dx": L.mortar_dense_linear_dx, "dw": L.mortar_dense_linear_dw}[form]
    _lib.check(fn(*head, TYPES[t], c.data_ptr(), c.stride(0), ws.data_ptr(), _stream()), form)
    Pd, Qd = P.double(), Q.double()
    exact = {"y": lambda: Qd @ Pd.t(), "dx": lambda: Qd @ Pd, "dw": lambda: Qd.t() @ Pd}[form]()
    intact = bool(cw[M:].isnan().all()) and bool(cw[:M, N:].isnan().all())
    return c, exact, intact


SIZES = [(65, 8, 8), (66, 24, 40), (128, 256, 64), (129, 264, 72), (200, 328, 200), (257, 520, 1000), (70, 64, 4096), (300, 128, 2736), (513, 1040, 136), (1030, 2064, 328)]


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("form", ["y", "dx", "dw"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_products_of_integers_are_exact(dev, form, M, N, K, t):
    if form == "dw":
        M, K = (M + 7) // 8 * 8, K - 3 if K > 8 else K       # rows of dW are features, its sums run over any number of tokens
    for extra in (0, 8):
        c, exact, intact = _product(form, M, N, K, t, dev, M + N + K, extra)
        assert torch.equal(c, exact.to(t)), (form, M, N, K, extra)
        assert intact


# enough tiles for the large ones, and few of them with long sums (ranges of K)
@pytest.mark.parametrize("form,M,N,K", [("y", 4096, 2048, 192), ("dx", 2100, 4104, 320), ("dw", 2048, 4096, 333), ("dw", 768, 768, 5000), ("dx", 130, 512, 8192), ("y", 100, 264, 9000)])
def test_large_products_of_integers_are_exact(dev, form, M, N, K):
    c, exact, intact = _product(form, M, N, K, torch.bfloat16, dev, 5)
    assert torch.equal(c, exact.to(torch.bfloat16)) and intact


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 48, 64])
def test_few_rows_of_integers_are_exact(dev, M, t):
    for N, K in ((8, 8), (24, 72), (264, 1000), (1040, 2736)):
        for extra in (0, 8):
            c, exact, intact = _product("y", M, N, K, t, dev, M + N, extra)
            assert torch.equal(c, exact.to(t)) and intact, (M, N, K, extra)


def _values24(buf, M, n):
    """The values of the kept gate_up output: 16 upper bits [M, n], then 8 bits [M, n]."""
    hi, lo = buf[:2 * M * n].view(torch.int16).int() << 16, buf[2 * M * n:3 * M * n].int() << 8
    return (hi | lo).view(torch.float32).view(M, n).double()


def _bytes24(v):
    bits = v.float().contiguous().view(torch.int32)
    return torch.cat([(bits >> 16).to(torch.int16).view(-1).view(torch.uint8), ((bits >> 8) & 0xff).to(torch.uint8).view(-1)])


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("M,d,f", [(1, 8, 8), (5, 64, 40), (16, 136, 264), (33, 1000, 72), (64, 256, 512), (65, 8, 8), (130, 72, 200), (300, 264, 136), (1100, 128, 1032)])
def test_gate_up_of_integers(dev, M, d, f, t):
    """The stored g and u exact, h the product of the unrounded ones: eight fp32 steps (exponential, reciprocal, three products) and one rounding."""
    L = _lib.lib()
    x, w = ints((M, d), 1, M, t, dev), ints((2 * f, d), 1, f, t, dev)
    hw, h = _padded(M, f, 8, t, dev)
    gu = torch.full((6 * M * f + 16,), 0xAB, dtype=torch.uint8, device=dev)
    for want_gu in (True, False):
        _lib.check(L.mortar_dense_gateup_swiglu(x.data_ptr(), M, d, d, w.data_ptr(), d, f, TYPES[t], h.data_ptr(), h.stride(0), gu.data_ptr() if want_gu else None,
                                                _stream()), "gateup")
        exact = x.double() @ w.double().t()
        g, u = exact.chunk(2, 1)
        ref = g * torch.sigmoid(g) * u
        assert_within(h, ref, rounding(t, ref) + 8 * 2.0 ** -23 * ref.abs(), "h")
        if want_gu:
            assert torch.equal(_values24(gu, M, 2 * f), exact) and bool((gu[6 * M * f:] == 0xAB).all())
            h.fill_(float("nan"))
        assert bool(hw[M:].isnan().all() and hw[:M, f:].isnan().all())


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("M,d,f", [(1, 8, 8), (7, 72, 40), (65, 200, 136), (300, 136, 264), (1100, 128, 1032)])
def test_swiglu_gradient_in_the_epilogue(dev, M, d, f, t):
    """dh exact (integers), gate and up as stored: the derivative and h to ten fp32 steps and one rounding."""
    L = _lib.lib()
    dy, w = ints((M, d), 1, M, t, dev), ints((d, f), 1, f, t, dev)
    gu = normals((M, 2 * f), 3, torch.float32, dev, 2.0)
    gu = (gu.view(torch.int32) & ~0xff).view(torch.float32)
    kept = _bytes24(gu)
    ow, dgu = _padded(M, 2 * f, 8, t, dev)
    hw, h = _padded(M, f, 8, t, dev)
    _lib.check(L.mortar_dense_swiglu_bwd(dy.data_ptr(), M, d, d, w.data_ptr(), f, f, TYPES[t], kept.data_ptr(), dgu.data_ptr(), dgu.stride(0), h.data_ptr(),
                                         h.stride(0), _stream()), "swiglu_bwd")
    dh = dy.double() @ w.double()
    g, u = gu.double().chunk(2, 1)
    s = torch.sigmoid(g)
    step = 10 * 2.0 ** -23
    ref = torch.cat([dh * u * s * (1 + g * (1 - s)), dh * g * s], 1)
    size = torch.cat([(dh * u).abs() * (s + (g * s * (1 - s)).abs()), (dh * g * s).abs()], 1)       # s + g s (1 - s) may cancel
    assert_within(dgu, ref, rounding(t, ref) + step * size, "dgu")
    assert_within(h, g * s * u, rounding(t, g * s * u) + step * (g * s * u).abs(), "h")
    assert bool(ow[M:].isnan().all() and ow[:M, 2 * f:].isnan().all() and hw[M:].isnan().all() and hw[:M, f:].isnan().all())


def _case(M, d, f, t, dev, seed, n=None):
    return (normals((M, d), seed, t, dev), normals((2 * f, d), seed + 1, t, dev, d ** -0.5), normals((n or d, f), seed + 2, t, dev, f ** -0.5),
            normals((M, n or d), seed + 3, t, dev))


def _grads(x, wgu, wd, dy):
    leaves = [v.detach().requires_grad_(True) for v in (x, wgu, wd)]
    y = ops.dense_mlp(*leaves)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


@pytest.mark.parametrize("t", list(TYPES), ids=str)
@pytest.mark.parametrize("M,d,f,n", [(1, 64, 128, None), (3, 8, 8, 16), (37, 256, 320, None), (64, 200, 88, 72), (65, 136, 264, None), (333, 768, 1024, None), (1500, 264, 136, 512)])
def test_mlp_and_gradients(dev, M, d, f, n, t):
    x, wgu, wd, dy = _case(M, d, f, t, dev, M + d, n)
    got, want, bounds = _grads(x, wgu, wd, dy), mlp_reference(x, wgu, wd, dy), mlp_bounds(x, wgu, wd, dy)
    for name, g, r, e in zip(("y", "dx", "dw_gate_up", "dw_down"), got, want, bounds):
        assert g.dtype == t
        assert_within(g, r, e, name)
    with torch.no_grad():
        assert torch.equal(ops.dense_mlp(x, wgu, wd), got[0])


def test_errors_are_those_of_rounding(dev):
    """Root mean square errors, where single wrong terms would show: a rounding to bf16 is off by 2^-9 / sqrt(3) relative on average at
    most; y and dw_down see the roundings of h and their own, dx and dw_gate_up those of dgu and their own."""
    x, wgu, wd, dy = _case(700, 512, 768, torch.bfloat16, dev, 5)
    one = 2.0 ** -9 * 2 / 3 ** 0.5
    for g, r, n in zip(_grads(x, wgu, wd, dy), mlp_reference(x, wgu, wd, dy), (2, 2, 2, 2)):
        assert float((g.double() - r).norm() / r.norm()) <= one * n ** 0.5


def test_gradient_against_differences(dev):
    """fp16 MLP along a direction: the loss <dy, y> at x +- e v against dx; each y is off by its bound at most, the quotient by e^2 times a third derivative."""
    x, wgu, wd, dy = _case(9, 64, 96, torch.float16, dev, 13)
    _, dx, _, _ = _grads(x, wgu, wd, dy)
    v, e = ints(x.shape, 1, 4, torch.float16, dev), 2.0 ** -3
    xp, xm = (x.float() + e * v.float()).half(), (x.float() - e * v.float()).half()
    real = (xp.double() - xm.double())                      # the step that was taken, roundings of x included
    with torch.no_grad():
        lp, lm = (float((dy.double() * ops.dense_mlp(p, wgu, wd).double()).sum()) for p in (xp, xm))
    noise = float((dy.abs().double() * (mlp_bounds(xp, wgu, wd) + mlp_bounds(xm, wgu, wd))).sum())
    want = float((dx.double() * real).sum())
    curved = abs(float((dy.double() * (mlp_reference(xp, wgu, wd) - mlp_reference(xm, wgu, wd))).sum()) - float((mlp_reference(x, wgu, wd, dy)[1] * real).sum()))
    assert abs((lp - lm) - want) <= noise + curved + float((mlp_bounds(x, wgu, wd, dy)[1] * real.abs()).sum())


def test_only_the_gradients_that_are_wanted(dev):
    case = _case(130, 136, 200, torch.bfloat16, dev, 17)
    full = _grads(*case)
    for i in range(3):
        leaves = [v.detach().requires_grad_(i == j) for j, v in enumerate(case[:3])]
        (g,) = torch.autograd.grad(ops.dense_mlp(*leaves), [leaves[i]], case[3])
        assert torch.equal(g, full[i + 1])


def test_shapes_and_strides(dev):
    x, wgu, wd, dy = _case(24, 64, 72, torch.bfloat16, dev, 19)
    y = ops.dense_mlp(x, wgu, wd)
    assert torch.equal(ops.dense_mlp(x.view(2, 3, 4, 64), wgu, wd), y.view(2, 3, 4, 64)) and torch.equal(ops.dense_mlp(x[0], wgu, wd), ops.dense_mlp(x[:1], wgu, wd)[0])
    wide = torch.full((24, 200), float("nan"), dtype=torch.bfloat16, device=dev)
    for view in (wide[:, 8:72], wide[:, 3:67], wide[:, 64:192:2]):
        view.copy_(x)
        assert torch.equal(ops.dense_mlp(view, wgu, wd), y)
    assert torch.equal(ops.dense_mlp(x.t().contiguous().t(), wgu, wd), y)
    assert torch.equal(ops.dense_mlp(x, wgu.t().contiguous().t(), wd.t().contiguous().t()), y)
    full = _grads(x, wgu, wd, dy)
    leaves = [x.view(2, 12, 64).detach().requires_grad_(True), wgu.t().contiguous().t().requires_grad_(True), wd.detach().requires_grad_(True)]
    got = torch.autograd.grad(ops.dense_mlp(*leaves), leaves, dy.view(2, 12, 64).transpose(0, 1).contiguous().transpose(0, 1))
    for g, w in zip(got, full[1:]):
        assert torch.equal(g.reshape(w.shape), w)
    rep = torch.ones((), dtype=torch.bfloat16, device=dev).expand(24, 64)
    (g,) = torch.autograd.grad(ops.dense_mlp(leaves[0].view(24, 64), wgu, wd), [leaves[0]], rep)
    assert_within(g.view(24, 64), mlp_reference(x, wgu, wd, rep)[1], mlp_bounds(x, wgu, wd, rep)[1], "dx of an expanded dy")


def test_no_rows(dev):
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=dev, requires_grad=True)
    _, wgu, wd, _ = _case(1, 64, 40, torch.bfloat16, dev, 1)
    wgu.requires_grad_(True), wd.requires_grad_(True)
    y = ops.dense_mlp(x, wgu, wd)
    gx, gg, gd = torch.autograd.grad(y, [x, wgu, wd], torch.empty_like(y))
    assert y.shape == gx.shape == (0, 64) and not gg.any() and not gd.any() and gg.shape == wgu.shape and gd.shape == wd.shape


def test_rows_stay_apart(dev):
    """A row with NaN or infinities leaves the others' bits alone, also in the tiles' tails."""
    x, wgu, wd, _ = _case(70, 72, 88, torch.bfloat16, dev, 23)
    for rows in (70, 20):
        good = ops.dense_mlp(x[:rows], wgu, wd)
        bad = x[:rows].clone()
        bad[3, 1], bad[rows - 1, 71] = float("nan"), float("inf")
        y = ops.dense_mlp(bad, wgu, wd)
        keep = [i for i in range(rows) if i not in (3, rows - 1)]
        assert torch.equal(y[keep], good[keep]) and bool(y[3].isnan().all())


def test_same_bits_on_another_stream_and_from_a_graph(dev):
    case = _case(400, 256, 320, torch.bfloat16, dev, 29)
    first = _grads(*case)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = _grads(*case)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(first, other))
    leaves, dy = [v.clone().requires_grad_(True) for v in case[:3]], case[3].clone()

    def step():
        y = ops.dense_mlp(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):                       # two graphs alive at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(3):
        new = _case(400, 256, 320, torch.bfloat16, dev, 90 + i)
        with torch.no_grad():
            for a, c in zip((*leaves, dy), new):
                a.copy_(c)
        want = _grads(*new)
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_refusals(dev):
    x, wgu, wd, _ = _case(4, 64, 72, torch.bfloat16, dev, 1)
    with pytest.raises(TypeError):
        ops.dense_mlp(x.float(), wgu, wd)
    with pytest.raises(TypeError):
        ops.dense_mlp(x, wgu.half(), wd)
    with pytest.raises(ValueError):
        ops.dense_mlp(x[:, :56], wgu, wd)
    with pytest.raises(ValueError):
        ops.dense_mlp(x, wgu[:136], wd)
    with pytest.raises(ValueError):
        ops.dense_mlp(x[:, :60], wgu[:, :60], wd)
    with pytest.raises(ValueError):
        ops.dense_mlp(x, wgu, wd[:60])
    with pytest.raises(RuntimeError):
        ops.dense_mlp(x, wgu.cpu(), wd)
    xl = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(ops.dense_mlp(xl, wgu, wd).sum(), [xl], create_graph=True)
