"""Rows, codes and gradients whose offsets pass 32 bits, looked at in places spread over all of them."""
import math

import pytest
import torch

from dense_util import assert_within, normals, rounding
from mortar_amd import ops
from operators_util import int4_bound, int4_weight, unpack_codes

pytestmark = pytest.mark.gpu
T = torch.bfloat16


def _places(n, count, dev):
    """`count` indices below n, its ends and those around 2^31 bytes and values of rows of any length among them."""
    return torch.linspace(0, n - 1, count, dtype=torch.float64).round().long().unique().to(dev)


def test_int4_results(dev):
    M, N, K = 66000, 33000, 64
    assert M * N > 1 << 31
    x = normals((M, K), 0, T, dev)
    c, s, z = ops.quantize_int4_weight(normals((N, K), 1, T, dev), 64, True)
    y = ops.linear_int4(x, c, s, z, 64)
    at = _places(M, 300, dev)
    ref = x[at].double() @ int4_weight(c, s, z, 64, K).t()
    assert_within(y[at], ref, int4_bound(x[at], s, z, 64, T, ref), "y")


@pytest.mark.parametrize("K", [1040, 1039])
def test_int4_rows_of_x(dev, K):
    M, N = 1100000, 24
    assert M * K * 2 > 1 << 31
    x = normals((1100, K), 0, T, dev).repeat(1000, 1)
    x += torch.arange(M, device=dev, dtype=torch.float32).div(M).to(T).unsqueeze(1)
    c, s, _ = ops.quantize_int4_weight(normals((N, K), 1, T, dev, K ** -0.5), 128)
    y = ops.linear_int4(x, c, s)
    at = _places(M, 2000, dev)
    ref = x[at].double() @ int4_weight(c, s, None, 128, K).t()
    assert_within(y[at], ref, int4_bound(x[at], s, None, 128, T, ref), "y")


@pytest.mark.parametrize("M", [1, 12, 200])
def test_int4_codes(dev, M):
    N, K = 530000, 8192
    assert N * K // 2 > 1 << 31
    c = torch.randint(-(1 << 31), 1 << 31, (N, K // 8), generator=torch.Generator(dev).manual_seed(0), device=dev, dtype=torch.int32)
    s = torch.rand((K // 128, N), generator=torch.Generator(dev).manual_seed(1), device=dev).t() * 0.01
    x = normals((M, K), 3, T, dev)
    y = ops.linear_int4(x, c, s)
    at = _places(N, 2000, dev)
    ref = x.double() @ int4_weight(c[at], s[at], None, 128, K).t()
    assert_within(y[:, at], ref, int4_bound(x, s[at], None, 128, T, ref), "y")


def test_int4_quantising(dev):
    N, K = 270000, 8192
    assert N * K > 1 << 31
    w = normals((100, K), 0, T, dev).repeat(N // 100, 1)
    c, s, _ = ops.quantize_int4_weight(w, 128)
    one, os, _ = ops.quantize_int4_weight(w[:100], 128)
    at = _places(N, 3000, dev)
    assert torch.equal(c[at], one[at % 100]) and torch.equal(s[at], os[at % 100]) and int(unpack_codes(one, K).max()) == 15


def test_rows_by_slot(dev):
    N, k, d = 33000, 8, 8200
    assert N * k * d > 1 << 31
    ids = torch.randint(0, 70, (N, k), generator=torch.Generator().manual_seed(0)).to(dev)
    order = ops.expert_sort(ids, 64)
    x, w = normals((N, d), 1, T, dev), normals((N, k), 2, torch.float32, dev)
    full = int(order.offsets[-1])
    xs = ops.expert_dispatch(x, order)
    at = _places(N * k, 4000, dev)
    assert torch.equal(xs[at], torch.where((at < full).unsqueeze(1), x[order.token[at].long()], torch.zeros((), dtype=T, device=dev)))
    w.requires_grad_(), xs.requires_grad_()
    y = ops.expert_combine(xs, w, order)
    dys, dw = torch.autograd.grad(y, (xs, w), x)
    place = _places(N, 500, dev)
    rows, live = order.position[place].long(), ids[place] < 64
    wl = torch.where(live, w.detach()[place], 0.0).double()
    ref, dot = wl.sum(1, keepdim=True) * x[place].double(), torch.where(live, (x[place].double() ** 2).sum(1, keepdim=True), 0.0)
    size = wl.abs().sum(1, keepdim=True) * x[place].double().abs()
    assert_within(y[place].detach(), ref, (k + 1) * 2.0 ** -24 * size + rounding(T, ref), "y")
    assert_within(dw[place], dot, (d // 64 + 20) * 2.0 ** -24 * dot + rounding(torch.float32, dot), "dw")
    want = wl.unsqueeze(2) * x[place].double().unsqueeze(1)
    assert_within(dys[rows], want, 2.0 ** -24 * want.abs() + rounding(T, want), "dys")


def test_one_gradient(dev):
    n = (1 << 31) + 12345
    g = torch.zeros(n, dtype=T, device=dev)
    at = _places(n, 5000, dev)
    g[at] = normals((at.numel(),), 0, T, dev)
    ref = float(g[at].double().norm())
    out = torch.full((n,), 7.0, dtype=torch.float32, device=dev)
    (got,), norm = ops.clip_grads([g], 0.5 * ref, out=[out])
    c = 0.5 * ref / (ref + 1e-6)
    want = g[at].double() * c
    assert abs(float(norm) - ref) <= 2.0 ** -24 * 1.001 * ref and float(ops.grad_norm([g], math.inf)) == float(g[at].abs().max())
    assert_within(got[at], want, 2.1 * 2.0 ** -24 * want.abs() + rounding(torch.float32, want), "result")
    assert int(torch.count_nonzero(got)) == int(torch.count_nonzero(want))
    ops.clip_grads([g], 0.5 * ref, out=[g])
    assert_within(g[at], want, 2.1 * 2.0 ** -24 * want.abs() + rounding(T, want), "in place")
