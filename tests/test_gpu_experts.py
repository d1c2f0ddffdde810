"""Tokens sorted by expert and back: the order and the dispatch exactly, sums and gradients within fp32 rounding per addition."""
import pytest
import torch

from dense_util import U32, assert_within, normals, rounding
from mortar_amd import ops
from operators_util import draw_ids, expert_order

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("N,k,E", [(1, 1, 1), (1, 8, 16), (3, 2, 5), (64, 1, 2), (100, 7, 9), (1000, 4, 64), (2048, 2, 63), (4096, 1, 1024), (4097, 1, 1), (5000, 3, 1023), (9000, 8, 352),
                                   (16384, 8, 64), (70000, 2, 1024), (200000, 1, 3)])
def test_order(dev, N, k, E, wide):
    ids = draw_ids(N, k, E, N + k + E, repeat=N * E > 1 << 21)
    if wide:
        ids = ids.long()
        ids[0, 0] = (1 << 40) + (0 if E > 1 else 5)                 # an empty slot, whatever its low bits say
        ids[-1, -1] = E
    order = ops.expert_sort(ids.to(dev), E)
    for got, want in zip(order, expert_order(ids, E)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("N", [10, 6000])
def test_orders_with_one_expert_or_none(dev, N):
    for ids in (torch.full((N, 2), -1), torch.full((N, 2), 3), torch.arange(2 * N).view(N, 2) % 4 + 0):
        for t in (torch.int32, torch.int64):
            for view in (ids.to(t).to(dev), ids.t().contiguous().to(t).to(dev).t()):
                for got, want in zip(ops.expert_sort(view, 4), expert_order(ids, 4)):
                    assert torch.equal(got.cpu(), want)
    empty = ops.expert_sort(torch.empty((0, 2), dtype=torch.int32, device=dev), 4)
    assert empty.position.shape == (0, 2) and empty.token.shape == (0,) and empty.offsets.tolist() == [0] * 5


SHAPES = [(1, 1, 1, 1), (1, 8, 16, 2048), (5, 3, 4, 7), (33, 2, 8, 64), (40, 9, 16, 1999), (129, 5, 352, 257), (700, 8, 64, 768), (64, 20, 32, 4100), (3, 2, 2, 40000)]


def _case(dev, N, k, E, d, t, wt, seed=0):
    ids = draw_ids(N, k, E, seed + N).to(dev)
    x, ys, dxs = (normals(s, seed + i, t, dev) for i, s in enumerate(((N, d), (N * k, d), (N * k, d))))
    dy, w = normals((N, d), seed + 4, t, dev), normals((N, k), seed + 5, wt, dev)
    return ids, x, ys, dxs, dy, w


def _reference(ids, E, x, ys, dxs, dy, w):
    position, token, offsets = (v.to(ids.device) for v in expert_order(ids.cpu(), E))
    full = ((ids >= 0) & (ids < E)).unsqueeze(2)
    rows = torch.arange(ys.shape[0], device=ids.device).unsqueeze(1) < offsets[-1]
    p = position.long()
    zero = torch.zeros((), dtype=torch.float64, device=ids.device)
    pick = torch.where(full, ys.double()[p], zero)
    wd = torch.where(full, w.double().unsqueeze(2), zero)
    r = {"xs": torch.where(rows, x.double()[token.long()], zero), "y": (wd * pick).sum(1), "y_size": (wd * pick).abs().sum(1)}
    g = torch.where(full, dxs.double()[p], zero)
    r["dx"], r["dx_size"] = g.sum(1), g.abs().sum(1)
    r["dys"] = torch.empty_like(r["xs"])
    r["dys"][p.view(-1)] = (wd * dy.double().unsqueeze(1)).view(-1, x.shape[1])
    dot = pick * dy.double().unsqueeze(1)
    r["dw"], r["dw_size"] = dot.sum(2), dot.abs().sum(2)
    return r


def _compare(got, r, k, d, t, wt):
    xs, y, dx, dys, dw = got
    assert torch.equal(xs.double(), r["xs"])
    assert_within(y, r["y"], (k + 1) * U32 * r["y_size"] + rounding(t, r["y"]), "y")
    assert_within(dx, r["dx"], (k + 1) * U32 * r["dx_size"] + rounding(t, r["dx"]), "dx")
    assert_within(dys, r["dys"], U32 * r["dys"].abs() + rounding(t, r["dys"]), "dys")
    assert_within(dw, r["dw"], (d // 64 + 20) * U32 * r["dw_size"] + rounding(wt, r["dw"]), "dw")


@pytest.mark.parametrize("t,wt", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)],
                         ids=str)
@pytest.mark.parametrize("N,k,E,d", SHAPES)
def test_there_and_back_with_gradients(dev, N, k, E, d, t, wt):
    ids, x, ys, dxs, dy, w = _case(dev, N, k, E, d, t, wt)
    r = _reference(ids, E, x, ys, dxs, dy, w)
    order = ops.expert_sort(ids, E)
    for v in (x, ys, w):
        v.requires_grad_(True)
    xs, y = ops.expert_dispatch(x, order), ops.expert_combine(ys, w, order)
    dx, dys, dw = torch.autograd.grad((xs, y), (x, ys, w), (dxs, dy))
    assert xs.dtype == y.dtype == dx.dtype == dys.dtype == t and dw.dtype == wt
    _compare((xs.detach(), y.detach(), dx, dys, dw), r, k, d, t, wt)
    with torch.no_grad():
        assert torch.equal(ops.expert_dispatch(x, order), xs) and torch.equal(ops.expert_combine(ys, w, order), y)
    plain = ops.expert_combine(ys, None, order)
    one = ops.expert_combine(ys, torch.ones_like(w), order)
    assert torch.equal(plain, one) and torch.equal(torch.autograd.grad(plain, ys, dy)[0], torch.autograd.grad(one, ys, dy)[0])


def test_empty_slots_are_not_looked_at(dev):
    """NaN in the rows and weights of empty slots goes nowhere; tokens without experts are 0."""
    for t in TYPES:
        ids, x, ys, dxs, dy, w = _case(dev, 60, 4, 8, 520, t, torch.float32, 3)
        ids[7] = -1
        order = ops.expert_sort(ids, 8)
        full = int(order.offsets[-1])
        r = _reference(ids, 8, x, ys, dxs, dy, w)
        ys[full:], dxs[full:] = float("nan"), float("nan")
        w[ids < 0] = float("nan")
        for v in (x, ys, w):
            v.requires_grad_(True)
        xs, y = ops.expert_dispatch(x, order), ops.expert_combine(ys, w, order)
        dx, dys, dw = torch.autograd.grad((xs, y), (x, ys, w), (dxs, dy))
        _compare((xs.detach(), y.detach(), dx, dys, dw), r, 4, 520, t, torch.float32)
        assert bool((y[7] == 0).all()) and bool((dx[7] == 0).all()) and bool((dw[ids < 0] == 0).all()) and bool((dys[full:] == 0).all())


def test_an_expert_twice(dev):
    """A token whose slots name one expert twice has two rows there."""
    ids = torch.tensor([[1, 1, 0], [0, 0, 0]], device=dev)
    order = ops.expert_sort(ids, 2)
    assert order.position.tolist() == [[4, 5, 0], [1, 2, 3]] and order.offsets.tolist() == [0, 4, 6] and order.token.tolist() == [0, 1, 1, 1, 0, 0]
    x = normals((2, 40), 0, torch.float32, dev).requires_grad_()
    (dx,) = torch.autograd.grad(ops.expert_dispatch(x, order).sum(), x)
    assert torch.equal(dx, torch.full_like(dx, 3.0))                 # (a broadcast gradient)


def test_strides(dev):
    """Rows apart, transposed, on odd addresses, one row for all tokens."""
    ids, x, ys, dxs, dy, w = _case(dev, 30, 3, 5, 77, torch.bfloat16, torch.float32, 9)
    order = ops.expert_sort(ids, 5)
    xs, y = ops.expert_dispatch(x, order), ops.expert_combine(ys, w, order)
    wide = torch.zeros((30, 99), dtype=x.dtype, device=dev)
    wide[:, 3:80] = x
    assert torch.equal(ops.expert_dispatch(wide[:, 3:80], order), xs) and torch.equal(ops.expert_dispatch(x.t().contiguous().t(), order), xs)
    assert torch.equal(ops.expert_dispatch(x[:1].expand(30, 77), order), ops.expert_dispatch(x[:1].repeat(30, 1), order))
    far = torch.zeros((90, 80), dtype=x.dtype, device=dev)
    far[:, 1:78] = ys
    wt = w.t().contiguous().t()
    assert torch.equal(ops.expert_combine(far[:, 1:78], wt, order), y)
    other = ops.ExpertOrder(order.position.t().contiguous().t(), order.token, order.offsets)
    assert torch.equal(ops.expert_combine(ys, w, other), y) and torch.equal(ops.expert_dispatch(x, other), xs)
    ys.requires_grad_(), wt.requires_grad_()
    g = wide[:, 5:82].copy_(dy)
    a = torch.autograd.grad(ops.expert_combine(ys, wt, other), (ys, wt), g)
    b = torch.autograd.grad(ops.expert_combine(ys, wt, order), (ys, wt), dy)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_gradients_against_differences(dev):
    """The result is linear in the rows and in the weights: differences are the derivative, up to fp32 rounding of sums of d k values on each side."""
    ids, x, ys, dxs, dy, w = _case(dev, 50, 4, 8, 100, torch.float32, torch.float32, 11)
    order = ops.expert_sort(ids, 8)
    vy, vw = normals((200, 100), 20, torch.float32, dev), normals((50, 4), 21, torch.float32, dev)
    ys.requires_grad_(), w.requires_grad_(), x.requires_grad_()
    dys, dw = torch.autograd.grad(ops.expert_combine(ys, w, order), (ys, w), dy)
    f = lambda a, b: float((ops.expert_combine(a, b, order).double() * dy.double()).sum())
    size = float((ops.expert_combine(ys.detach().abs() + vy.abs(), w.detach().abs() + vw.abs(), order).double() * dy.double().abs()).sum())
    with torch.no_grad():
        assert abs(f(ys + vy, w) - f(ys - vy, w) - 2 * float((dys.double() * vy.double()).sum())) <= 40 * U32 * size
        assert abs(f(ys, w + vw) - f(ys, w - vw) - 2 * float((dw.double() * vw.double()).sum())) <= 40 * U32 * size
    (dx,) = torch.autograd.grad(ops.expert_dispatch(x, order), x, dxs)
    with torch.no_grad():                                            # <dispatch(v), dxs> = <v, dx>
        v = normals((50, 100), 22, torch.float32, dev)
        left, right = (ops.expert_dispatch(v, order).double() * dxs.double()), (v.double() * dx.double())
        assert abs(float(left.sum() - right.sum())) <= 8 * U32 * float(left.abs().sum())


def test_parts_of_the_gradient(dev):
    """Only what is asked for, and no tokens at all."""
    ids, x, ys, dxs, dy, w = _case(dev, 20, 3, 4, 72, torch.bfloat16, torch.float32, 5)
    order = ops.expert_sort(ids, 4)
    both = torch.autograd.grad(ops.expert_combine(ys.requires_grad_(), w.requires_grad_(), order), (ys, w), dy)
    only = torch.autograd.grad(ops.expert_combine(ys, w.detach(), order), ys, dy) + torch.autograd.grad(ops.expert_combine(ys.detach(), w, order), w, dy)
    assert torch.equal(only[0], both[0]) and torch.equal(only[1], both[1])
    none = ops.expert_sort(ids[:0], 4)
    x0, y0, w0 = (v.detach()[:0].requires_grad_() for v in (x, ys, w))
    for out, ins in ((ops.expert_dispatch(x0, none), (x0,)), (ops.expert_combine(y0, w0, none), (y0, w0))):
        assert out.shape == (0, 72) and all(g.numel() == 0 for g in torch.autograd.grad(out.sum(), ins))
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(ops.expert_combine(ys, w, order).float().sum(), ys, create_graph=True)


def test_refusals(dev):
    ids, x, ys, dxs, dy, w = _case(dev, 20, 3, 4, 72, torch.bfloat16, torch.float32, 5)
    order = ops.expert_sort(ids, 4)
    bad_order = ops.ExpertOrder(order.position.long(), order.token, order.offsets)
    for bad in (lambda: ops.expert_sort(ids, 0), lambda: ops.expert_sort(ids, 1025), lambda: ops.expert_sort(ids[0], 4), lambda: ops.expert_sort(ids[:, :0], 4), lambda: ops.expert_dispatch(x[:19], order),
                lambda: ops.expert_dispatch(x[0], order), lambda: ops.expert_dispatch(x[:, :0], order), lambda: ops.expert_combine(ys[:-1], w, order), lambda: ops.expert_combine(ys, w[:, :2], order),
                lambda: ops.expert_combine(ys, w, ops.ExpertOrder(order.position, order.token, order.offsets[:1]))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.expert_sort(ids.float(), 4), lambda: ops.expert_sort(ids, "4"), lambda: ops.expert_dispatch(x.double(), order), lambda: ops.expert_dispatch(x, bad_order),
                lambda: ops.expert_combine(ys, w.double(), order)):
        with pytest.raises(TypeError):
            bad()


def test_rows_that_no_cache_holds(dev):
    """Rows by slot of 268 MB and more, which are stored past the caches."""
    N, k, E, d = 8200, 8, 16, 1024
    ids, x, ys, dxs, dy, w = _case(dev, N, k, E, d, torch.float32, torch.float32, 2)
    assert N * k * d * 4 > 256 << 20
    order = ops.expert_sort(ids, E)
    full = int(order.offsets[-1])
    xs = ops.expert_dispatch(x, order)
    assert torch.equal(xs[:full], x[order.token[:full].long()]) and bool((xs[full:] == 0).all())
    (dys,) = torch.autograd.grad(ops.expert_combine(ys.requires_grad_(), w, order), ys, dy)
    want = torch.zeros_like(ys.detach()).index_copy_(0, order.position.view(-1).long(), torch.where(ids < 0, 0.0, w).unsqueeze(2).mul(dy.unsqueeze(1)).view(-1, d))
    assert torch.equal(dys, want)


def test_positions_outside_are_left_out(dev):
    """An order whose positions are none of its rows writes and reads nothing there."""
    ids, x, ys, dxs, dy, w = _case(dev, 20, 3, 4, 72, torch.float32, torch.float32, 5)
    good = ops.expert_sort(ids.clamp(min=0), 4)
    position = good.position.clone()
    position[3, 1], position[4, 2], position[5, 0] = 60, -1, 1 << 30
    order = ops.ExpertOrder(position, good.token, good.offsets)
    out = ops.expert_combine(ys, w, order)
    hole = w.clone()
    hole[3, 1] = hole[4, 2] = hole[5, 0] = 0
    assert torch.equal(out, ops.expert_combine(ys, hole, good))
    ops.expert_dispatch(x, order)
    large = ops.ExpertOrder(good.position, good.token, good.offsets + 1000)
    assert torch.equal(ops.expert_combine(ys, w, large), ops.expert_combine(ys, w, good))


@pytest.mark.parametrize("N", [3, 3000])
def test_captured(dev, N):
    """A captured step with its backward: every replay is the eager result."""
    ids, x, ys, dxs, dy, w = _case(dev, N, 3, 8, 136, torch.bfloat16, torch.float32, 1)
    leaves = [v.requires_grad_() for v in (x, ys, w)]

    def step():
        order = ops.expert_sort(ids, 8)
        xs, y = ops.expert_dispatch(x, order), ops.expert_combine(ys, w, order)
        return (*order, xs.detach(), y.detach(), *torch.autograd.grad((xs, y), leaves, (dxs, dy)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (5, 6, 7):
        new = _case(dev, N, 3, 8, 136, torch.bfloat16, torch.float32, seed)
        with torch.no_grad():
            for a, b in zip((ids, x, ys, dxs, dy, w), new):
                a.copy_(b)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("N,k,E", [(150000, 2, 40), (600000, 1, 7), (150001, 4, 1024), (1200, 1000, 64)])
def test_order_of_many_slots(dev, N, k, E):
    """Runs of more slots per lane, and of more workgroups than one batch of their counts."""
    ids = draw_ids(N, k, E, N, repeat=True).to(dev)
    order = ops.expert_sort(ids, E)
    key = torch.where((ids >= 0) & (ids < E), ids, E).view(-1)
    key, rows = torch.sort(key, stable=True)
    assert torch.equal(order.token, (rows // k).int())
    assert torch.equal(order.position.view(-1)[rows], torch.arange(N * k, dtype=torch.int32, device=dev))
    assert torch.equal(order.offsets, torch.searchsorted(key, torch.arange(E + 1, dtype=key.dtype, device=dev)).int())


@pytest.mark.parametrize("N,k,E,d", [(9, 70, 80, 264), (5, 130, 200, 77), (2, 64, 64, 520)])
@pytest.mark.parametrize("t,wt", [(torch.bfloat16, torch.float32), (torch.float32, torch.float16)], ids=str)
def test_more_slots_than_lanes(dev, N, k, E, d, t, wt):
    ids, x, ys, dxs, dy, w = _case(dev, N, k, E, d, t, wt)
    r = _reference(ids, E, x, ys, dxs, dy, w)
    order = ops.expert_sort(ids, E)
    for v in (x, ys, w):
        v.requires_grad_(True)
    xs, y = ops.expert_dispatch(x, order), ops.expert_combine(ys, w, order)
    dx, dys, dw = torch.autograd.grad((xs, y), (x, ys, w), (dxs, dy))
    _compare((xs.detach(), y.detach(), dx, dys, dw), r, k, d, t, wt)


@pytest.mark.parametrize("k", [1, 2, 3, 4])
@pytest.mark.parametrize("N", [1, 2, 3, 5, 6, 7])
def test_tokens_that_share_a_wave(dev, N, k):
    """Few slots per token: waves of several tokens, the last of them with fewer."""
    ids, x, ys, dxs, dy, w = _case(dev, N, k, 6, 100, torch.bfloat16, torch.float32, 40 + k)
    r = _reference(ids, 6, x, ys, dxs, dy, w)
    y = ops.expert_combine(ys, w, ops.expert_sort(ids, 6))
    assert_within(y, r["y"], (k + 1) * U32 * r["y_size"] + rounding(torch.bfloat16, r["y"]), "y")
