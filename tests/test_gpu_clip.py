"""The norm over many gradients and their clipping, against 64 bits: the norm and the factor are 64-bit values rounded to fp32, a product is rounded to fp32 and to its type."""
import math

import pytest
import torch

from dense_util import U32, assert_within, normals, rounding
from mortar_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _norm(grads, norm_type=2.0):
    d = [g.double().reshape(-1) for g in grads if g.numel()]
    if not d:
        return 0.0
    return max(float(v.abs().max()) for v in d) if norm_type == math.inf else math.sqrt(math.fsum(float((v * v).sum()) for v in d))


def _check(grads, results, norm, max_norm, norm_type=2.0, inputs=None):
    ref = _norm(inputs or grads, norm_type)
    assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - ref) <= U32 * 1.001 * ref
    c = min(1.0, max_norm / (ref + 1e-6))
    for i, (g, r) in enumerate(zip(inputs or grads, results)):
        v = g.double() * c
        assert_within(r, v, rounding(r.dtype, v) + 2.1 * U32 * v.abs(), f"result {i}")


def _many(sizes, seed, dev, types):
    flat = {t: normals((sum(sizes) + 16,), seed + i, t, dev) for i, t in enumerate(types)}
    out, at = [], 0
    for i, n in enumerate(sizes):
        out.append(flat[types[i % len(types)]][at:at + n])
        at += n
    return out


CASES = [([1], TYPES[:1]), ([7], TYPES[1:2]), ([0, 5, 0], TYPES[2:]), ([8192], TYPES[:1]), ([8191, 8193, 4096, 4095, 1], TYPES), ([3 * 8192 + 11] * 5, TYPES), ([1, 2, 3, 4, 5, 6, 7, 8, 9] * 60, TYPES),
         ([17] * 128, TYPES), ([1000] * 129, TYPES[:2]), ([1 << 22, 5, 777777], TYPES), ([11, 40000] * 200, TYPES[1:])]


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("sizes,types", CASES, ids=[str(i) for i in range(len(CASES))])
def test_clipping(dev, sizes, types, norm_type):
    """Flat buffers cut into tensors on odd addresses; factors below and at 1; results in the type, in fp32, in place."""
    grads = _many(sizes, len(sizes), dev, types)
    before = [g.clone() for g in grads]
    top = _norm(grads, norm_type)
    norm = ops.grad_norm(grads, norm_type)
    assert abs(float(norm) - top) <= U32 * 1.001 * top
    for max_norm in (0.3 * top, 2 * top, 0.0):
        got, n = ops.clip_grads(grads, max_norm, norm_type)
        _check(grads, got, n, max_norm, norm_type)
        assert torch.equal(n, norm) and all(g.dtype == r.dtype for g, r in zip(grads, got))
    got, n = ops.clip_grads(grads, 0.3 * top, norm_type, out=[torch.empty_like(g, dtype=torch.float32) for g in grads])
    _check(grads, got, n, 0.3 * top, norm_type)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    got, n = ops.clip_grads(grads, 0.3 * top, norm_type, out=grads)
    _check(before, grads, n, 0.3 * top, norm_type)
    assert all(a is b for a, b in zip(got, grads))


def test_neighbours_are_left_alone(dev):
    """Results lie between other values of the same 16 bytes."""
    flat = normals((1000,), 0, torch.bfloat16, dev)
    keep = flat.clone()
    parts = [flat[3:10], flat[11:500], flat[501:999]]
    ops.clip_grads(parts, 0.1, out=parts)
    assert torch.equal(flat[[0, 1, 2, 10, 500, 999]], keep[[0, 1, 2, 10, 500, 999]])
    _check(parts, parts, ops.grad_norm([keep[3:10], keep[11:500], keep[501:999]]), 0.1, inputs=[keep[3:10], keep[11:500], keep[501:999]])


def test_parameters(dev):
    """Parameters as a model has them: one without a gradient, one twice, a gradient with other strides, one that is a part of a larger one; versions go on."""
    a, b, c, d = (torch.nn.Parameter(torch.zeros(s, device=dev)) for s in ((40, 30), (7,), (9, 8), (6, 5)))
    a.grad, c.grad = normals((40, 30), 1, torch.float32, dev), normals((8, 9), 2, torch.float32, dev).t()
    d.grad = normals((6, 11), 3, torch.float32, dev)[:, 2:7]
    old = [p.grad.clone() for p in (a, c, d)]
    versions = [p.grad._version for p in (a, c, d)]
    norm = ops.clip_grad_norm_([a, b, c, a, d, d], 0.5)
    _check(None, [p.grad for p in (a, c, d)], norm, 0.5, inputs=old)
    assert b.grad is None and all(p.grad._version > v for p, v in zip((a, c, d), versions))
    assert float(ops.clip_grad_norm_(a, 100.0)) == pytest.approx(float(a.grad.norm()), rel=1e-6)
    now = a.grad.clone()
    ops.clip_grad_norm_((p for p in [a]), 100.0)                 # an iterator; a factor of 1 changes nothing
    assert torch.equal(a.grad, now)


def test_torch_agrees(dev):
    ps = [torch.nn.Parameter(torch.zeros(s, device=dev)) for s in ((100, 30), (77,), (1,))]
    for norm_type in (2.0, math.inf):
        for i, p in enumerate(ps):
            p.grad = normals(tuple(p.shape), i, torch.float32, dev)
        mine = ops.clip_grad_norm_(ps, 0.7, norm_type=norm_type)
        got = [p.grad.clone() for p in ps]
        for i, p in enumerate(ps):
            p.grad = normals(tuple(p.shape), i, torch.float32, dev)
        theirs = torch.nn.utils.clip_grad_norm_(ps, 0.7, norm_type=norm_type)
        torch.testing.assert_close(mine, theirs, rtol=1e-6, atol=0)
        torch.testing.assert_close(got, [p.grad for p in ps], rtol=1e-6, atol=0)


@pytest.mark.parametrize("value,types", [(1e30, [torch.float32, torch.bfloat16]), (1e-30, [torch.float32, torch.bfloat16]), (6e4, [torch.float16]), (6e-8, [torch.float16]),
                                         (1e-44, [torch.float32])])
def test_ends_of_the_range(dev, value, types):
    """Squares that fp32 cannot hold."""
    grads = [torch.full((500,), value, dtype=t, device=dev) for t in types]
    ref = _norm(grads)
    norm = ops.grad_norm(grads)
    assert ref > 0 and abs(float(norm) - ref) <= U32 * 1.001 * ref + 2.0 ** -150
    got, _ = ops.clip_grads(grads, ref / 4)
    c = min(1.0, ref / 4 / (ref + 1e-6))
    for g, r in zip(grads, got):
        v = g.double() * c
        assert_within(r, v, rounding(r.dtype, v) + 2.1 * U32 * v.abs() + 2.0 ** -150, "result")


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("t", TYPES, ids=str)
def test_values_that_are_not_finite(dev, t, norm_type):
    """An infinite norm makes the finite gradients 0, NaN all of them NaN."""
    for bad in (math.inf, -math.inf, math.nan):
        g = [normals((9000,), 0, t, dev), normals((3,), 1, t, dev)]
        g[0][8999] = bad
        got, norm = ops.clip_grads(g, 1.0, norm_type)
        if math.isnan(bad):
            assert math.isnan(norm) and all(bool(torch.isnan(r).all()) for r in got)
        else:
            assert float(norm) == math.inf and bool((got[0][:8999] == 0).all()) and bool((got[1] == 0).all()) and bool(torch.isnan(got[0][8999]))
        p = torch.nn.Parameter(torch.zeros(9000, dtype=t, device=dev))
        p.grad = g[0].clone()
        with pytest.raises(RuntimeError, match="not finite"):
            ops.clip_grad_norm_([p], 1.0, norm_type, error_if_nonfinite=True)
        assert torch.equal(p.grad[:8999], g[0][:8999])


def test_same_bits_every_time(dev):
    grads = _many([100000, 3, 77, 2500000], 5, dev, TYPES)
    first = ops.grad_norm(grads)
    assert all(torch.equal(ops.grad_norm(grads), first) for _ in range(5))


def test_overlapping_results_are_refused(dev):
    f = normals((100,), 0, torch.float32, dev)
    h = normals((100,), 0, torch.bfloat16, dev)
    keep = f.clone()
    for grads, out in (([f, f], [f, f]), ([f[:60], f[40:]], [f[:60], f[40:]]), ([f[:50], f[50:]], [f[50:], f[:50]]), ([f[:50]], [f[10:60]]),
                       ([f[:10], f[20:30]], [f[50:60], f[55:65]]), ([h[:20]], [h.view(torch.float32)[:20]]), ([f[:10]], [f[:1].expand(10)])):
        with pytest.raises(ValueError, match="overlap|several times"):
            ops.clip_grads(grads, 1.0, out=out)
    m = f.view(10, 10)
    with pytest.raises(ValueError, match="overlap"):
        ops.clip_grads([f, m[:, :3]], 1.0, out=[f, m[:, :3]])
    assert torch.equal(f, keep)
    got, n = ops.clip_grads([f, f], 1e9)                          # read twice, counted twice
    assert abs(float(n) - math.sqrt(2) * _norm([f])) < 1e-5 and torch.equal(got[0], f) and torch.equal(got[1], f)
    halves = [m[:, 0::2], m[:, 1::2]]                             # interleaved, in place
    ops.clip_grads(halves, 1.0, out=halves)
    _check(None, [f], ops.grad_norm([keep]), 1.0, inputs=[keep])


def test_refusals(dev):
    f = normals((10,), 0, torch.float32, dev)
    for bad in (lambda: ops.clip_grads([f], -1.0), lambda: ops.clip_grads([f], math.nan), lambda: ops.clip_grads([f], 1.0, norm_type=1), lambda: ops.clip_grads([f], 1.0, out=[]),
                lambda: ops.clip_grads([f], 1.0, out=[f[:5]])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.grad_norm([f.double()]), lambda: ops.grad_norm([f, None]), lambda: ops.clip_grads([f], 1.0, out=[f.half()]), lambda: ops.clip_grads([f], "1")):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.grad_norm([f.clone().requires_grad_()])
    with pytest.raises(RuntimeError, match="strided"):
        ops.grad_norm([f.to_sparse()])


def test_captured(dev):
    grads = _many([5000, 3, 20000, 64] * 40, 1, dev, TYPES)
    out = [torch.empty_like(g) for g in grads]
    ops.clip_grads(grads, 1.0, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm = ops.clip_grads(grads, 1.0, out=out)
    for seed in (7, 8, 9):
        for g, new in zip(grads, _many([5000, 3, 20000, 64] * 40, seed, dev, TYPES)):
            g.copy_(new)
        graph.replay()
        eager, n = ops.clip_grads(grads, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(eager, out))


@pytest.mark.parametrize("tensors", [300, 620])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_many_launches(dev, norm_type, tensors):
    """More partial sums than the clipping adds in every workgroup; results that go past the caches."""
    grads = _many([70000] * tensors, 4, dev, [torch.bfloat16, torch.float32])
    before = [g.clone() for g in grads]
    top = _norm(grads, norm_type)
    got, n = ops.clip_grads(grads, 0.4 * top, norm_type)
    _check(grads, got, n, 0.4 * top, norm_type)
    got, again = ops.clip_grads(grads, 0.4 * top, norm_type, out=grads)
    assert torch.equal(n, again) and torch.equal(n, ops.grad_norm(before, norm_type))
    _check(before, grads, n, 0.4 * top, norm_type)


def test_tensors_of_inference_mode(dev):
    """Writing them is refused outside of it, as torch's own calls do, with nothing written."""
    with torch.inference_mode():
        g = normals((100,), 0, torch.float32, dev)
        ops.clip_grads([g], 1.0, out=[g])
        keep = g.clone()
    with pytest.raises(RuntimeError, match="inference"):
        ops.clip_grads([g], 0.1, out=[g])
    assert torch.equal(g, keep)
    assert torch.allclose(ops.clip_grads([g], 0.1)[0][0], keep * 0.1, rtol=1e-5)
