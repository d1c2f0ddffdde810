"""Calls at the edges of the 4-bit layer, clipping and the expert rows: weights that are zeros, the end of the range of x, orders with slots taken
out, recomputed forwards, strided results that share memory."""
import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from dense_util import assert_within, normals
from mortar_amd import ops
from operators_util import draw_ids, int4_bound, int4_weight, pack_codes

pytestmark = pytest.mark.gpu


# ---- 4-bit layers


#: rows, outputs, inputs, group: products of few rows (x through LDS, as operands, 32 rows of x) and tiles of both sizes, in one and several ranges of K
ZERO_FORMS = [(1, 40, 2048, 128), (3, 40, 1024, 64), (13, 264, 5632, 32), (7, 520, 1999, 128), (40, 264, 1040, 64), (17, 8200, 1040, 32), (300, 2055, 8200, 128), (4200, 264, 264, 32),
              (4200, 131, 4104, 64), (4200, 131, 4099, 128), (6000, 517, 131, 32), (6000, 517, 136, 128), (2000, 520, 6152, 32)]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M,N,K,group", ZERO_FORMS)
def test_weights_of_zero_add_nothing(dev, M, N, K, group, t, zeros):
    """Rows of zeros give exactly 0, and what x holds where a group of weights is zeros does not change a bit."""
    w = normals((N, K), N, torch.float32, dev, 1e-4).to(t)
    first, last = slice(0, group), slice((K - 1) // group * group, K)
    w[1], w[N - 2] = 0, 0
    w[2:20, first], w[20:36, last] = 0, 0
    c, s, z = ops.quantize_int4_weight(w, group, zeros)
    x = normals((M, K), M, t, dev, 8.0)
    y = ops.linear_int4(x, c, s, z, group)
    assert bool((y[:, [1, N - 2]] == 0).all()) and bool((y[:, 0] != 0).any())
    for rows, part in ((slice(2, 20), first), (slice(20, 36), last)):
        other = x.clone()
        other[:, part] = normals(tuple(other[:, part].shape), 3, t, dev, 100.0)
        assert torch.equal(ops.linear_int4(other, c, s, z, group)[:, rows], y[:, rows])
    other = x.clone()
    other[:, first] = 0
    ref = other[:, :].double() @ int4_weight(c, s, z, group, K).t()
    got = ops.linear_int4(other, c, s, z, group)
    assert_within(got[:, 2:20], ref[:, 2:20], int4_bound(other, s[2:20], None if z is None else z[2:20], group, t, ref[:, 2:20]), "y")


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M,N,K,group", ZERO_FORMS)
def test_codes_at_their_zero_points_add_nothing(dev, M, N, K, group, t):
    """The same for codes of a caller's own, whatever the zero point and the scale."""
    g = torch.Generator().manual_seed(K)
    groups = -(-K // group)
    z = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8).to(dev)
    s = (torch.rand((N, groups), generator=g) + 0.5).to(dev)
    at = z.long().repeat_interleave(group, 1)[:, :K]
    q = torch.randint(0, 16, (N, K), generator=g).to(dev)
    zero = torch.rand((N, groups), generator=g).to(dev).round().bool().repeat_interleave(group, 1)[:, :K]
    q[::3] = torch.where(zero, at, q)[::3]
    q[::4] = at[::4]
    x = normals((M, K), M, t, dev, 8.0)
    y = ops.linear_int4(x, pack_codes(q), s, z, group)
    assert bool((y[:, ::4] == 0).all())
    ref = x.double() @ int4_weight(pack_codes(q), s, z, group, K).t()
    assert_within(y, ref, int4_bound(x, s, z, group, t, ref), "y")


@pytest.mark.parametrize("M,N,K,group", [(1, 40, 2048, 128), (7, 520, 1999, 64), (40, 264, 1040, 32), (4200, 264, 264, 128), (6000, 517, 136, 32), (4200, 131, 4104, 64)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=str)
def test_zero_points_beyond_the_codes(dev, M, N, K, group, t):
    """Zero points take 8 bits: W = (c - z) s also where z is more than any code."""
    groups = -(-K // group)
    g = torch.Generator().manual_seed(N)
    z = torch.randint(0, 256, (N, groups), generator=g, dtype=torch.uint8).to(dev)
    z[0], z[1], z[2], z[3] = 255, 16, 15, 241
    q = torch.randint(0, 16, (N, K), generator=g).to(dev)
    s = torch.full((N, groups), 2.0 ** -6, dtype=t, device=dev)
    x = normals((M, K), M, t, dev)
    ref = x.double() @ int4_weight(pack_codes(q), s, z, group, K).t()
    assert_within(ops.linear_int4(x, pack_codes(q), s, z, group), ref, int4_bound(x, s, z, group, t, ref), "y")


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 40, 2048), (7, 520, 1999), (40, 264, 1040), (4200, 264, 264), (6000, 517, 136)])
def test_large_activations(dev, M, N, K, group, zeros):
    """The end of the documented range: 32 times a group's sum of |x| just below the largest fp32 number."""
    limit = torch.finfo(torch.float32).max / 32
    w = normals((N, K), 5, torch.bfloat16, dev, 2.0 ** -6)
    w[0] = 0
    c, s, z = ops.quantize_int4_weight(w, group, zeros)
    x = torch.zeros((M, K), dtype=torch.bfloat16, device=dev)
    x[0, 3], x[0, K - 1] = 0.995 * limit, -0.995 * limit            # alone in their groups
    if M > 1:
        x[1] = 0.99 * limit / group                                  # all of one sign
    y = ops.linear_int4(x, c, s, z, group)
    ref = x.double() @ int4_weight(c, s, z, group, K).t()
    assert bool((y[:, 0] == 0).all())
    assert_within(y, ref, int4_bound(x, s, z, group, torch.bfloat16, ref), "y")


@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("K,wide", [(5640, 8192), (5632, 5640), (2560, 4096), (2048, 2056), (1040, 1536)])
@pytest.mark.parametrize("M", [2, 5, 8, 13, 16])
def test_rows_of_x_apart(dev, M, K, wide, group):
    """Few rows of a wider buffer: the rows' distance chooses how x is read, and nothing else."""
    buffer = torch.full((M, wide), float("nan"), dtype=torch.bfloat16, device=dev)
    x = buffer[:, :K].copy_(normals((M, K), M, torch.bfloat16, dev))
    c, s, _ = ops.quantize_int4_weight(normals((136, K), K, torch.bfloat16, dev, K ** -0.5), group)
    ref = x.double() @ int4_weight(c, s, None, group, K).t()
    for v in (x, x.contiguous()):
        assert_within(ops.linear_int4(v, c, s, group_size=group), ref, int4_bound(x, s, None, group, torch.bfloat16, ref), "y")


# ---- expert rows


def _soil(*shapes, dtype, dev):
    """Memory that the next allocations of these shapes take holds NaN."""
    held = [torch.full(s, float("nan"), dtype=dtype, device=dev) for s in shapes for _ in range(3)]
    torch.cuda.synchronize()
    del held


def _taken_out(N, k, dev):
    """(order, the same with some positions that are none of its rows, which slots those are)"""
    ids = draw_ids(N, k, 9, N, repeat=True).to(dev)
    good = ops.expert_sort(ids, 9)
    out = torch.rand((N, k), generator=torch.Generator().manual_seed(6)).to(dev) < 0.3
    out[0, 0], out[N - 1] = True, True
    bad = torch.tensor([-1, N * k, 1 << 30, -(1 << 31)], dtype=torch.int32, device=dev)[torch.arange(N * k, device=dev).view(N, k) % 4]
    return good, ops.ExpertOrder(torch.where(out, bad, good.position), good.token, good.offsets), out


TAKEN_OUT = [(20, 3, 72), (300, 8, 520), (9, 70, 77), (700, 1, 1999)]


@pytest.mark.parametrize("t,wt", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.float16)], ids=str)
@pytest.mark.parametrize("N,k,d", TAKEN_OUT)
def test_slots_taken_out_have_no_gradient(dev, N, k, d, t, wt):
    """Positions that are none of the rows (slots dropped behind the sort) are empty slots: their weights have a gradient of 0, the others theirs."""
    good, order, out = _taken_out(N, k, dev)
    dy, w, ys = normals((N, d), 2, t, dev), normals((N, k), 3, wt, dev), normals((N * k, d), 4, t, dev)
    ys.requires_grad_(), w.requires_grad_()
    _soil((N, k), dtype=wt, dev=dev)
    (dw,) = torch.autograd.grad(ops.expert_combine(ys.detach(), w, order), w, dy)
    (want,) = torch.autograd.grad(ops.expert_combine(ys.detach(), w, good), w, dy)
    assert torch.equal(dw, torch.where(out, 0, want))
    dys, dw = torch.autograd.grad(ops.expert_combine(ys, w, order), (ys, w), dy)
    hole = torch.where(out, 0, w.detach())
    rows = good.position[~out].long()
    assert torch.equal(dw, torch.where(out, 0, want)) and torch.equal(dys[rows], torch.autograd.grad(ops.expert_combine(ys, hole, good), ys, dy)[0][rows])


@pytest.mark.parametrize("t,wt", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.float16)], ids=str)
@pytest.mark.parametrize("named", [True, False])
@pytest.mark.parametrize("N,k,d", TAKEN_OUT)
def test_rows_without_a_slot_are_zeros(dev, N, k, d, t, wt, named):
    """Rows whose slots were taken out, in what is dispatched and in the gradient of the combined rows; an order of a caller's own may have no tokens."""
    good, order, out = _taken_out(N, k, dev)
    order = order if named else order._replace(token=None)
    x, dy, w, ys = (normals(s, i, v, dev) for i, (s, v) in enumerate((((N, d), t), ((N, d), t), ((N, k), wt), ((N * k, d), t))))
    gone = torch.zeros((N * k, 1), dtype=torch.bool, device=dev)
    gone[good.position[out].long()] = True
    x.requires_grad_(), ys.requires_grad_(), w.requires_grad_()
    _soil((N * k, d), dtype=t, dev=dev)
    xs = ops.expert_dispatch(x, order)
    assert torch.equal(xs.detach(), torch.where(gone, 0, ops.expert_dispatch(x.detach(), good)))
    (dx,) = torch.autograd.grad(xs, x, ys.detach())
    assert torch.equal(dx, torch.autograd.grad(ops.expert_dispatch(x, good), x, torch.where(gone, 0, ys.detach()))[0])
    y = ops.expert_combine(ys, w, order)
    hole = torch.where(out, 0, w.detach())
    want = ops.expert_combine(ys, hole, good)
    _soil((N * k, d), dtype=t, dev=dev)
    dys, dw = torch.autograd.grad(y, (ys, w), dy)
    assert torch.equal(y, want) and torch.equal(dys, torch.autograd.grad(want, ys, dy)[0])
    plain = ops.expert_combine(ys, None, order)
    _soil((N * k, d), dtype=t, dev=dev)
    one = ops.expert_combine(ys, torch.where(out, 0, torch.ones_like(w)).detach(), good)
    assert torch.equal(plain, one) and torch.equal(torch.autograd.grad(plain, ys, dy)[0], torch.autograd.grad(one, ys, dy)[0])


def test_tokens_of_an_order_are_checked(dev):
    order = ops.expert_sort(draw_ids(20, 3, 4, 0).to(dev), 4)
    x = normals((20, 16), 0, torch.float32, dev)
    for token, error in ((order.token[:-1], ValueError), (order.token.view(20, 3), ValueError), (order.token.long(), TypeError), (order.token.cpu(), RuntimeError)):
        with pytest.raises(error, match="token|ROCm"):
            ops.expert_dispatch(x, order._replace(token=token))
        with pytest.raises(error, match="token|ROCm"):
            ops.expert_combine(x.repeat(3, 1), None, order._replace(token=token))


@pytest.mark.parametrize("named", [False, True])
def test_recomputed_forward(dev, named):
    """The forward run again inside a backward that names its inputs saves what the first one did."""
    ids = draw_ids(40, 3, 5, 0).to(dev)
    order = ops.expert_sort(ids, 5)
    x, dy, scores = (normals(s, i, torch.float32, dev) for i, s in enumerate(((40, 64), (40, 64), (40, 3))))
    x.requires_grad_(), scores.requires_grad_()

    def block(x, scores):
        xs = ops.expert_dispatch(x, order)
        return ops.expert_combine(xs * xs, torch.softmax(scores, dim=1), order)

    want = torch.autograd.grad(block(x, scores), (x, scores), dy)
    y = checkpoint(block, x, scores, use_reentrant=False)
    if named:
        got = torch.autograd.grad(y, (x, scores), dy)
    else:
        y.backward(dy)
        got = x.grad, scores.grad
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- clipping


def test_strided_results_that_share_memory_are_refused(dev):
    """Results that do not lie as their gradients do, too, share memory neither with each other nor with another gradient."""
    f = normals((20, 24), 0, torch.float32, dev)
    a, b = normals((20, 3), 1, torch.float32, dev), normals((20, 3), 2, torch.float32, dev)
    r, keep = torch.full((20, 24), 7.0, device=dev), f.clone()
    square = [normals((8, 8), i, torch.float32, dev) for i in (3, 4)]
    o = torch.zeros((8, 8), device=dev)
    for grads, out in (([a, b], [r[:, :3], r[:, :3]]), ([a, b], [r[:, :3], r[:, 2:5]]), ([a, b], [r[:, 1:4], r[:, 0:6:2]]), ([square[0].t(), square[1].t()], [o, o]),
                       ([square[0].t(), square[1]], [o, o]), ([a, f[:, :3]], [f[:, :3], r[:, :3]]), ([a, f], [f[:, 4:7], r]), ([a, b], [r[:, :3], r.view(-1)[480 - 62:480 - 2].view(20, 3)]),
                       ([a, b[:10]], [r[:, :3], r[::2, 2:5]]), ([a, b], [r[:, :3], r.as_strided((20, 3), (23, 1))]),
                       ([f[:, :3], a], [f[:, 1:4], r[:, :3]]), ([f[:, :3], a], [r[:, :3], f.view(-1)[24:84].view(20, 3)]), ([f[:, 0:6:2], a], [r[:, 5:8], f[:, 2:5]])):
        with pytest.raises(ValueError, match="overlap"):
            ops.clip_grads(grads, 1.0, out=out)
    assert bool((r == 7).all()) and torch.equal(f, keep)
    with pytest.raises(ValueError, match="overlap"):                # in place: columns that two gradients share
        ops.clip_grads([f[:, :3], f[:, 2:5]], 1.0, out=[f[:, :3], f[:, 2:5]])
    ps = [torch.nn.Parameter(torch.zeros(20, 3, device=dev)) for _ in range(2)]
    ps[0].grad, ps[1].grad = f[:, :3], f[:, 2:5]
    with pytest.raises(ValueError, match="overlap"):
        ops.clip_grad_norm_(ps, 1.0)
    assert torch.equal(f, keep)


def test_strided_results_side_by_side(dev):
    """Slices of one matrix that share nothing are taken: columns, every other column, rows and columns of other distances, a row between the columns of another."""
    a, b = normals((20, 3), 1, torch.float32, dev), normals((20, 3), 2, torch.float32, dev)
    c = min(1.0, 1.0 / (math.sqrt(float((a.double() ** 2).sum() + (b.double() ** 2).sum())) + 1e-6))

    def check(grads, out, views):
        r = torch.full((20, 24), 7.0, device=dev)
        keep = r.clone()
        o = [v(r) for v in views]
        ops.clip_grads(grads, 1.0, out=o)
        for v, g in zip(o, grads):
            torch.testing.assert_close(v.double(), g.double() * c, rtol=1e-6, atol=0)
        mask = torch.zeros_like(r)
        for v in views:
            v(mask).fill_(1.0)
        assert torch.equal(torch.where(mask.bool(), keep, r), keep)

    check([a, b], None, [lambda r: r[:, :3], lambda r: r[:, 3:6]])
    check([a, b], None, [lambda r: r[:, 0:6:2], lambda r: r[:, 1:6:2]])
    check([a, b], None, [lambda r: r[:, 21:24], lambda r: r.as_strided((20, 3), (24, 8), 4)])
    check([a, b], None, [lambda r: r.view(40, 12)[0::2, :3], lambda r: r.view(40, 12)[1::2, :3]])
    one = normals((3,), 3, torch.float32, dev)
    r = torch.zeros((20, 24), device=dev)
    got, n = ops.clip_grads([a, one], 1e9, out=[r[:, :3], r[5, 8:11]])
    assert torch.equal(r[:, :3], a) and torch.equal(r[5, 8:11], one)
    halves = [r.copy_(normals((20, 24), 4, torch.float32, dev))[:, 0::2], r[:, 1::2]]
    keep, n = r.clone(), ops.grad_norm([r])
    ops.clip_grads(halves, 1.0, out=halves)
    torch.testing.assert_close(r, keep * (1.0 / (n + 1e-6)), rtol=1e-6, atol=0)
