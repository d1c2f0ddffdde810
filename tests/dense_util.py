"""Error bounds of the dense operators in 64 bits, and integer operands whose products are exact."""
import torch

U32 = 2.0 ** -24                                   # half a step of fp32, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}     # half the smallest step


def rounding(t, v):
    """Largest error of rounding the values v once to the type t."""
    return torch.finfo(t).eps / 2 * v.abs() + TINY[t]


def ints(shape, most, seed, dtype, device):
    """Integers -most .. most: sums of products below 2^24 are exact in fp32 in any order."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g).to(dtype).to(device)


def normals(shape, seed, dtype, device, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)


def assert_within(got, ref, bound, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), f"{what}: {int((~(err <= bound)).sum())} of {err.numel()} beyond the bound, worst {float((err / bound).max()):.2f} of it"


# ---- layer norm


def norm_reference(x, w, b, eps, dy=None):
    """(y, dx, dw, db) of the formulas in 64 bits."""
    x = x.double()
    w = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if w is None else w.double()
    c = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    z = c * r
    y = z * w + (0.0 if b is None else b.double())
    if dy is None:
        return y
    dy = dy.double()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - z * (g * z).mean(1, keepdim=True))
    return y, dx, (dy * z).sum(0), dy.sum(0)


def norm_bounds(x, w, b, eps, dy=None):
    """Bounds of the same results when every fp32 operation rounds once.  A sum of n values adds at most `chain` of them one behind the
    other (values of a thread, then a tree of 8 and the division), so it is off by chain * U32 * sum |.|; what a quantity is off by
    enters whatever is formed from it to first order, doubled for the second."""
    t = x.dtype
    x = x.double()
    d = x.shape[1]
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    chain = 72 + d // 256 + 10
    u = U32 * chain
    mu = x.mean(1, keepdim=True)
    c = x - mu
    var = (c * c).mean(1, keepdim=True)
    r = 1.0 / torch.sqrt(var + eps)
    z = c * r
    e_mu = u * x.abs().mean(1, keepdim=True) + U32 * mu.abs()
    e_c = e_mu + U32 * (c.abs() + mu.abs())
    e_var = u * var + 2 * (c.abs() * e_c).mean(1, keepdim=True)
    e_r = r * (0.5 * e_var * r * r + 4 * U32)
    e_z = e_c * r + c.abs() * e_r + U32 * z.abs()
    y = z * w + b
    e_y = 2 * (e_z * w.abs() + 2 * U32 * ((z * w).abs() + b.abs())) + rounding(t, y)
    if dy is None:
        return e_y
    dy = dy.double()
    g = dy * w
    e_g = U32 * g.abs()
    e1 = e_g.mean(1, keepdim=True) + u * g.abs().mean(1, keepdim=True)
    s2 = (g * z).mean(1, keepdim=True)
    e2 = (e_g * z.abs() + g.abs() * e_z).mean(1, keepdim=True) + u * (g * z).abs().mean(1, keepdim=True)
    s1 = g.mean(1, keepdim=True)
    inner = g - s1 - z * s2
    e_inner = e_g + e1 + e_z * s2.abs() + z.abs() * e2 + 4 * U32 * (g.abs() + s1.abs() + (z * s2).abs())
    dx = r * inner
    e_dx = 2 * (r * e_inner + e_r * inner.abs() + U32 * dx.abs()) + rounding(t, dx)
    rows = U32 * (x.shape[0] / 512 + 512 / 16 + 32)
    e_dw = 2 * ((dy.abs() * e_z).sum(0) + rows * (dy * z).abs().sum(0))
    e_db = 2 * rows * dy.abs().sum(0)
    return e_y, e_dx, e_dw, e_db


# ---- dense mlp


def mlp_reference(x, wgu, wd, dy=None):
    x, wgu, wd = x.double(), wgu.double(), wd.double()
    g, u = (x @ wgu.t()).chunk(2, 1)
    s = torch.sigmoid(g)
    h = g * s * u
    y = h @ wd.t()
    if dy is None:
        return y
    dy = dy.double()
    dh = dy @ wd
    dgu = torch.cat([dh * u * s * (1 + g * (1 - s)), dh * g * s], 1)
    return y, dgu @ wgu, dgu.t() @ x, dy.t() @ h


def mlp_bounds(x, wgu, wd, dy=None):
    """Bounds of the same results: products exact, sums of K products off by K * U32 * sum |.|, silu and its derivative by 8 fp32 steps
    (exponential and reciprocal of the hardware, one step each), h and dgu rounded to 16 bits and g, u to 24 between the kernels,
    results rounded once.  |silu'| <= 1.1, |silu''| <= 0.5."""
    t = x.dtype
    x, wgu, wd = x.double(), wgu.double(), wd.double()
    d, f = wgu.shape[1], wd.shape[1]
    g, u = (x @ wgu.t()).chunk(2, 1)
    eg, eu = (U32 * d * (x.abs() @ wgu.abs().t())).chunk(2, 1)
    s = torch.sigmoid(g)
    si = g * s
    h = si * u
    e_h = u.abs() * (1.1 * eg + 8 * U32 * si.abs()) + si.abs() * eu + 2 * U32 * h.abs()
    y = h @ wd.t()
    e_y = 1.05 * ((rounding(t, h) + e_h) @ wd.abs().t() + U32 * f * (h.abs() @ wd.abs().t())) + rounding(t, y)
    if dy is None:
        return e_y
    dy = dy.double()
    n, M = dy.shape[1], x.shape[0]
    dh = dy @ wd
    e_dh = U32 * n * (dy.abs() @ wd.abs())
    eg, eu = eg + 2.0 ** -16 * g.abs(), eu + 2.0 ** -16 * u.abs()
    ds = s * (1 + g * (1 - s))
    e_si = 1.1 * eg + 8 * U32 * si.abs()
    e_ds = 0.5 * eg + 16 * U32
    du, dg = dh * si, dh * u * ds
    e_du = e_dh * si.abs() + dh.abs() * e_si + rounding(t, du)
    e_dg = e_dh * (u * ds).abs() + dh.abs() * (eu * ds.abs() + u.abs() * e_ds) + rounding(t, dg)
    dgu, e_dgu = torch.cat([dg, du], 1), 1.05 * torch.cat([e_dg, e_du], 1)
    e_h2 = 1.05 * (e_si * u.abs() + si.abs() * eu) + rounding(t, h)
    dx, dwgu, dwd = dgu @ wgu, dgu.t() @ x, dy.t() @ h
    e_dx = e_dgu @ wgu.abs() + U32 * 2 * f * (dgu.abs() @ wgu.abs()) + rounding(t, dx)
    e_dwgu = e_dgu.t() @ x.abs() + U32 * M * (dgu.abs().t() @ x.abs()) + rounding(t, dwgu)
    e_dwd = dy.abs().t() @ e_h2 + U32 * M * (dy.abs().t() @ h.abs()) + rounding(t, dwd)
    return e_y, 1.05 * e_dx, 1.05 * e_dwgu, 1.05 * e_dwd


# ---- 8 bits


def fp8_rows(x):
    """(codes as e4m3, scales [M, kb]) of the definition in torch operations."""
    m, k = x.shape
    kb = -(-k // 128)
    p = torch.zeros((m, kb * 128), dtype=torch.float32, device=x.device)
    p[:, :k] = x.float()
    p = p.view(m, kb, 128)
    a = p.abs().amax(2)
    s = torch.where(a > 0, a * torch.tensor(1.0 / 448.0, dtype=torch.float32, device=a.device), torch.ones_like(a))
    q = (p / s[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(m, kb * 128)[:, :k].contiguous()
    return q.view(torch.float8_e4m3fn), s


def fp8_weight(w):
    n, k = w.shape
    nb, kb = -(-n // 128), -(-k // 128)
    p = torch.zeros((nb * 128, kb * 128), dtype=torch.float32, device=w.device)
    p[:n, :k] = w.float()
    p = p.view(nb, 128, kb, 128)
    a = p.abs().amax((1, 3))
    s = torch.where(a > 0, a * torch.tensor(1.0 / 448.0, dtype=torch.float32, device=a.device), torch.ones_like(a))
    q = (p / s[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(nb * 128, kb * 128)[:n, :k].contiguous()
    return q.view(torch.float8_e4m3fn), s


def fp8_reference(xq, xs, wq, ws):
    """(y, bound) in 64 bits.  Inside one matrix instruction the products of a group of K values are aligned to the largest of them and
    cut 13 bits below it (measured: 2^8 + 2^-5 is kept, 2^8 + 2^-6 is not); 128 products of a block are each off by at most 2^-13 of
    the block's largest possible product.  Then one fp32 multiply-add per block, and the result's rounding."""
    n, k = wq.shape
    kb = -(-k // 128)
    x, w = xq.double(), wq.double()
    y = torch.zeros((x.shape[0], n), dtype=torch.float64, device=x.device)
    e = torch.zeros_like(y)
    total = torch.zeros_like(y)
    for b in range(kb):
        xb, wb = x[:, b * 128:(b + 1) * 128], w[:, b * 128:(b + 1) * 128]
        f = xs[:, b].double()[:, None] * ws[:, b].double().repeat_interleave(128)[:n][None, :]
        y += (xb @ wb.t()) * f
        total += (xb.abs() @ wb.abs().t()) * f
        e += 128 * 2.0 ** -13 * xb.abs().amax(1)[:, None] * wb.abs().amax(1)[None, :] * f
    return y, e + U32 * (kb + 4) * total + rounding(torch.bfloat16, y)
