"""Dense companions of the carved MLP as their users run them, one pass each through the public entry points.

  norm_forward   ops.layernorm on the rows of a batch, no gradients
  norm_train     the same with its backward pass: dx and the gradients of weight and bias
  mlp_forward    ops.dense_mlp: the SwiGLU MLP of a block that is not carved (yet), serving and evaluation
  mlp_train      the same with its backward pass: dx and the gradients of both weights
  fp8            ops.linear_fp8: a dense layer served in 8 bits, bf16 activations quantised in the call

Weights are U(-1, 1) / sqrt(in_features), as the layers initialise them; activations N(0, 1) behind a norm, with a few
louder features where they are quantised; what a norm is fed has rows of different size and features of different mean.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
E4M3_MAX = 448.0
GROUP = 128
MAX_MLP_FLOPS = 8.0e11      # of a drawn case: less than the largest listed one
MAX_NORM_VALUES = 1 << 25


def _norm(name, kind, rows, d, dtype):
    return {"name": name, "kind": kind, "rows": rows, "d": d, "dtype": dtype}


def _mlp(name, kind, rows, d, d_ff, dtype="bf16"):
    return {"name": name, "kind": kind, "rows": rows, "d": d, "d_ff": d_ff, "dtype": dtype}


def _fp8(name, rows, n_in, n_out):
    return {"name": name, "kind": "fp8", "rows": rows, "n_in": n_in, "n_out": n_out}


def listed():
    return [
        # the norm in front of one block for a few decoding streams: launch latency
        _norm("norm_forward_4", "norm_forward", 4, 2048, "bf16"),
        # the router's query norm in a training step at base width, 4 x 4096 tokens: fp32 rows
        _norm("norm_train_query", "norm_train", 16384, 768, "fp32"),
        # a block's norm in a training step at the benchmark's width
        _norm("norm_train_block", "norm_train", 16384, 2048, "bf16"),
        # an odd batch of rows of an odd width that no vector load fits
        _norm("norm_train_odd", "norm_train", 1021, 1999, "fp16"),
        # one token through an uncarved block at the benchmark's width: both weights are streamed once
        _mlp("mlp_forward_1", "mlp_forward", 1, 2048, 5632),
        # an odd batch of streams through the same block
        _mlp("mlp_forward_37", "mlp_forward", 37, 2048, 5632),
        # the benchmark's prompt through an uncarved block
        _mlp("mlp_forward_4096", "mlp_forward", 4096, 2048, 5632),
        # the training step before the carve at base width, 4 x 4096 tokens
        _mlp("mlp_train_base", "mlp_train", 16384, 768, 2048),
        # the training step before the carve at the benchmark's width: the largest case
        _mlp("mlp_train_4096", "mlp_train", 4096, 2048, 5632),
        # a ragged batch through a block whose widths fit no tile, in fp16
        _mlp("mlp_train_odd", "mlp_train", 1003, 1040, 2736, "fp16"),
        # one token through the gate_up layer of a block served in 8 bits
        _fp8("fp8_1", 1, 2048, 11264),
        # the benchmark's prompt through the same layer
        _fp8("fp8_4096", 4096, 2048, 11264),
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v // step * step))


def draw(rng):
    kind = rng.choice(["norm_forward", "norm_train", "mlp_forward", "mlp_train", "fp8"])
    rows = _log_int(rng, 1, 16384)
    if kind.startswith("norm"):
        d = _log_int(rng, 64, 8192, rng.choice([1, 8]))
        rows = max(1, min(rows, MAX_NORM_VALUES // d))
        return {"kind": kind, "rows": rows, "d": d, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "fp8":
        n_in, n_out = _log_int(rng, 256, 8192, 16), _log_int(rng, 256, 16384, 16)
        rows = max(1, min(rows, int(MAX_MLP_FLOPS / (2.0 * n_in * n_out))))
        return {"kind": kind, "rows": rows, "n_in": n_in, "n_out": n_out}
    d = _log_int(rng, 256, 4096, 16)
    d_ff = _log_int(rng, d, 3 * d, 16)
    flops = (6.0 if kind == "mlp_forward" else 18.0) * d * d_ff
    rows = max(1, min(rows, int(MAX_MLP_FLOPS / flops)))
    return {"kind": kind, "rows": rows, "d": d, "d_ff": d_ff, "dtype": rng.choice(["bf16", "fp16"])}


# ---------------------------------------------------------------------------------------------------- inputs


def _inputs(case, seed):
    """The tensors of a case, made from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def weight(n_out, n_in):
        return (torch.rand((n_out, n_in), generator=g, device="cuda") * 2 - 1) / math.sqrt(n_in)

    rows, kind = case["rows"], case["kind"]
    if kind == "fp8":
        loud = 1.0 + 15.0 * (torch.rand(case["n_in"], generator=g, device="cuda") < 0.01)
        return {"x": (normal(rows, case["n_in"]) * loud).bfloat16(), "w": weight(case["n_out"], case["n_in"]).bfloat16()}
    t, d = DTYPES[case["dtype"]], case["d"]
    if kind.startswith("norm"):
        size = 0.5 + 2.0 * torch.rand((rows, 1), generator=g, device="cuda")
        s = {"x": (normal(rows, d) * size + 0.5 * normal(d)).to(t), "weight": (1.0 + 0.1 * normal(d)).to(t), "bias": (0.1 * normal(d)).to(t)}
    else:
        s = {"x": normal(rows, d).to(t), "w_gate_up": weight(2 * case["d_ff"], d).to(t), "w_down": weight(d, case["d_ff"]).to(t)}
    if kind.endswith("train"):
        s["dy"] = normal(rows, d).to(t)
    return s


def _quantise_weight(w):
    """e4m3 values and one fp32 scale per 128 x 128 block: scale = amax / 448 (1 for a block of zeros), value = rne(w / scale)."""
    n, k = w.shape
    nb, kb = -(-n // GROUP), -(-k // GROUP)
    p = torch.zeros((nb * GROUP, kb * GROUP), dtype=torch.float32, device=w.device)
    p[:n, :k] = w.float()
    p = p.view(nb, GROUP, kb, GROUP)
    amax = p.abs().amax(dim=(1, 3))
    s = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    q = (p / s[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).view(nb * GROUP, kb * GROUP)[:n, :k].contiguous().view(torch.float8_e4m3fn), s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "fp8":
        s["wq"], s["ws"] = _quantise_weight(s.pop("w"))
    elif case["kind"].endswith("train"):
        for name, t in s.items():
            if name != "dy":
                t.requires_grad_(True)
    s["kind"] = case["kind"]
    return s


# ---------------------------------------------------------------------------------------------------- one pass


def _run_own(s):
    from mortar_amd import ops
    kind = s["kind"]
    if kind == "fp8":
        return ops.linear_fp8(s["x"], s["wq"], s["ws"])
    if kind.startswith("norm"):
        args = (s["x"], s["weight"], s["bias"])
        call = lambda: ops.layernorm(*args, eps=EPS)
    else:
        args = (s["x"], s["w_gate_up"], s["w_down"])
        call = lambda: ops.dense_mlp(*args)
    if kind.endswith("forward"):
        with torch.no_grad():
            return call()
    y = call()
    return (y.detach(), *torch.autograd.grad(y, args, s["dy"]))


def _quantise_rows(x, t):
    """The values that e4m3 with one scale per row and 128 features stands for, in the type t.  The quotient is an fp32 one by definition."""
    m, k = x.shape
    kb = -(-k // GROUP)
    p = torch.zeros((m, kb * GROUP), dtype=torch.float32, device=x.device)
    p[:, :k] = x.float()
    p = p.view(m, kb, GROUP)
    amax = p.abs().amax(dim=2, keepdim=True)
    sc = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    return ((p / sc).to(torch.float8_e4m3fn).to(t) * sc.to(t)).view(m, kb * GROUP)[:, :k]


def _weight_values(wq, ws, t):
    n, k = wq.shape
    return wq.to(t) * ws.to(t).repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]


@torch.no_grad()
def _run_plain(s):
    kind = s["kind"]
    if kind == "fp8":
        x = _quantise_rows(s["x"], torch.float32)
        w = _weight_values(s["wq"], s["ws"], torch.float32)
        return (x @ w.t()).bfloat16()
    x = s["x"].float()
    t = s["x"].dtype
    if kind.startswith("norm"):
        w, b = s["weight"].float(), s["bias"].float()
        c = x - x.mean(dim=1, keepdim=True)
        r = torch.rsqrt((c * c).mean(dim=1, keepdim=True) + EPS)
        xh = c * r
        y = xh * w + b
        if kind == "norm_forward":
            return y.to(t)
        dy = s["dy"].float()
        g = dy * w
        dx = r * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))
        return y.to(t), dx.to(t), (dy * xh).sum(dim=0).to(t), dy.sum(dim=0).to(t)
    wgu, wd = s["w_gate_up"].float(), s["w_down"].float()
    gate, up = (x @ wgu.t()).chunk(2, dim=1)
    sg = 1.0 / (1.0 + torch.exp(-gate))
    silu = gate * sg
    h = silu * up
    y = h @ wd.t()
    if kind == "mlp_forward":
        return y.to(t)
    dy = s["dy"].float()
    dh = dy @ wd
    dgu = torch.cat([dh * up * (sg + silu * (1.0 - sg)), dh * silu], dim=1)
    return y.to(t), (dgu @ wgu).to(t), (dgu.t() @ x).to(t), (dy.t() @ h).to(t)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------- definition


@torch.no_grad()
def exact(case, seed):
    """The definitions in 64 bits."""
    s = _inputs(case, seed)
    if case["kind"] == "fp8":
        wq, ws = _quantise_weight(s["w"])
        return _quantise_rows(s["x"], torch.float64) @ _weight_values(wq, ws, torch.float64).t()
    x = s["x"].double()
    if case["kind"].startswith("norm"):
        mean, var = x.mean(dim=1, keepdim=True), x.var(dim=1, unbiased=False, keepdim=True)
        sd = torch.sqrt(var + EPS)
        z = (x - mean) / sd
        y = z * s["weight"].double() + s["bias"].double()
        if case["kind"] == "norm_forward":
            return y
        dy = s["dy"].double()
        dz = dy * s["weight"].double()
        d = case["d"]
        dx = (dz - (dz.sum(dim=1, keepdim=True) + z * (dz * z).sum(dim=1, keepdim=True)) / d) / sd
        return y, dx, torch.einsum("ij,ij->j", dy, z), dy.sum(dim=0)
    wg, wu = s["w_gate_up"].double().split(case["d_ff"])
    wd = s["w_down"].double()
    a, b = x @ wg.t(), x @ wu.t()
    sig = torch.sigmoid(a)
    h = a * sig * b
    y = h @ wd.t()
    if case["kind"] == "mlp_forward":
        return y
    dy = s["dy"].double()
    dh = dy @ wd
    da, db = dh * b * sig * (1 + a * (1 - sig)), dh * a * sig
    return y, da @ wg + db @ wu, torch.cat([da.t() @ x, db.t() @ x]), dy.t() @ h


def work(case):
    """What no implementation can do without: every input read once, every output written once, the products' multiply-adds."""
    rows, kind = case["rows"], case["kind"]
    if kind == "fp8":
        k, n = case["n_in"], case["n_out"]
        scales = 4 * (-(-n // GROUP)) * (-(-k // GROUP))
        return {"bytes": 2 * rows * k + n * k + scales + 2 * rows * n, "flops": 2 * rows * n * k}
    e, d = (4 if case["dtype"] == "fp32" else 2), case["d"]
    train = kind.endswith("train")
    if kind.startswith("norm"):
        return {"bytes": e * ((4 if train else 2) * rows * d + (4 if train else 2) * d), "flops": (20 if train else 8) * rows * d}
    weights = 3 * d * case["d_ff"]
    return {"bytes": e * ((4 if train else 2) * rows * d + (2 if train else 1) * weights), "flops": (18 if train else 6) * rows * d * case["d_ff"]}
