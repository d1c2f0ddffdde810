"""The operators together, as a user runs them: router, tokens to experts, ops.dense_mlp per expert, back with the gates, backward, clipping, and the trained
weights served in 4 bits to single tokens."""
import pytest
import torch

from mortar_amd import TileRouter, ops
from operators_util import int4_weight

pytestmark = pytest.mark.gpu

E, K, D, F, N = 8, 3, 128, 256, 200


def _experts(xs, order, gu, dn):
    """Each expert's MLP on its rows; the rows behind the last expert's stay zeros."""
    at = order.offsets.tolist()
    parts = [ops.dense_mlp(xs[at[e]:at[e + 1]], gu[e], dn[e]) for e in range(E)]
    return torch.cat(parts + [xs.new_zeros((xs.shape[0] - at[E], D))])


def _plain(x, gates, gu, dn):
    """The same in 64 bits, every expert on every token."""
    y = torch.zeros_like(x)
    for e in range(E):
        g, u = (x @ gu[e].t()).chunk(2, dim=1)
        y = y + gates[:, e:e + 1] * ((torch.nn.functional.silu(g) * u) @ dn[e].t())
    return y


def test_a_routed_step_and_its_serving(dev):
    torch.manual_seed(0)
    router = TileRouter(E, D, activation_ratio=K / E).to(dev)
    x = torch.randn((N, D), device=dev).bfloat16().requires_grad_()
    gu = [(torch.randn((2 * F, D), device=dev) * D ** -0.5).bfloat16().requires_grad_() for _ in range(E)]
    dn = [(torch.randn((D, F), device=dev) * F ** -0.5).bfloat16().requires_grad_() for _ in range(E)]
    with torch.no_grad():
        gates, _ = router(x.float())
    gates = gates.float().requires_grad_()
    w, ids = gates.topk(K, dim=1)
    ids = ids.masked_fill(w <= 0, -1)
    assert bool((ids < 0).any())                                     # the threshold leaves slots empty
    order = ops.expert_sort(ids, E)
    ys = _experts(ops.expert_dispatch(x, order), order, gu, dn)
    y = ops.expert_combine(ys, w, order)
    dy = torch.randn((N, D), device=dev).bfloat16()
    leaves = [x, gates, *gu, *dn]
    grads = torch.autograd.grad(y, leaves, dy)

    wide = [v.detach().double().requires_grad_() for v in leaves]
    ref = _plain(wide[0], wide[1], wide[2:2 + E], wide[2 + E:])
    want = torch.autograd.grad(ref, wide, dy.double())
    # gates of inactive experts: the formula gives them a derivative, the slots none
    on = (gates > 0).double()
    want = [g * on if i == 1 else g for i, g in enumerate(want)]
    # bf16 between the launches: x, h, y of the expert, y and on the way back dy w, d(gate, up), dx of the expert: at most 8 roundings, 2^-8 each, one after the other
    y, ref = y.detach(), ref.detach()
    assert (y.double() - ref).norm() <= 4 * 2.0 ** -8 * ref.norm()
    for g, r in zip(grads, want):
        assert (g.double() - r).norm() <= 8 * 2.0 ** -8 * r.norm()           # (an expert that has no tokens: 0)

    for p, g in zip(gu + dn, grads[2:]):
        p.grad = g
    norm = ops.clip_grad_norm_(gu + dn, 0.5)
    assert float(norm) > 0.5
    # rounding to bf16 moves each value by at most 2^-8 of it, and so the norm
    assert abs(float(ops.grad_norm([p.grad for p in gu + dn])) - 0.5) <= 0.5 * 2.0 ** -8 + 1e-5
    with torch.no_grad():
        for p in gu + dn:
            p.add_(p.grad, alpha=-1.0)
        token = x[:1].detach()
        codes, scales, zeros = ops.quantize_int4_weight(gu[0], 64, True)
        served = ops.linear_int4(token, codes, scales, zeros, 64).double()
        exact = token.double() @ int4_weight(codes, scales, zeros, 64, D).t()
        assert float((served - exact).norm() / exact.norm()) <= 2.0 ** -8
        assert float((exact - token.double() @ gu[0].double().t()).norm() / exact.norm()) < 0.5


def test_serving_one_token_through_its_experts(dev):
    """The same calls for a single token, captured once and replayed: sort, dispatch, 4-bit products of the experts' rows, combine."""
    torch.manual_seed(1)
    x = torch.randn((1, D), device=dev).bfloat16()
    weights = [ops.quantize_int4_weight((torch.randn((D, D), device=dev) * D ** -0.5).bfloat16()) for _ in range(E)]
    ids = torch.tensor([[5, 0, -1]], dtype=torch.int32, device=dev)
    w = torch.tensor([[0.75, 0.25, float("nan")]], device=dev)

    def step():
        order = ops.expert_sort(ids, E)
        xs = ops.expert_dispatch(x, order)
        ys = torch.cat([ops.linear_int4(xs[i:i + 1], *weights[e]) for i, e in enumerate((0, 5))] + [xs[2:]])
        return ops.expert_combine(ys, w, order)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for seed in (1, 2, 3):
        x.copy_(torch.randn((1, D), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and bool(torch.isfinite(y).all())
