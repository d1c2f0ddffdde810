"""What a dense MLP needs around its products, as its users run it: one pass each through the public entry points.

  int4            ops.linear_int4: a dense layer served from 4-bit codes with one scale (and zero point) per row and group of inputs
  clip            ops.clip_grads: the norm over the gradients of many tensors, and the gradients clipped to it
  experts_forward ops.expert_sort, ops.expert_dispatch, ops.expert_combine: tokens to their experts' rows and back, serving
  experts_train   the same with the backward passes: gradients of the tokens, of the experts' results and of the weights

Weights are U(-1, 1) / sqrt(in_features) as the layers initialise them, activations N(0, 1).  Gradients are N(0, 1) with a size of their own per
tensor, views of one flat buffer per type, as bucketed training holds them.  A token's experts are different ones, the popular ones drawn more often,
with the weights of a router in front; some cases have empty slots (fewer experts than slots), as a router with a threshold leaves.
The experts' products lie between dispatch and combine and are not part of these calls: their results are among the inputs.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_INT4_FLOPS = 1.8e11     # of a drawn case: less than the largest listed one
MAX_ROUTED_VALUES = 1 << 25
MAX_GRADIENTS = 1 << 26
NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)       # where in its word the value j of each eight lies


def _int4(name, rows, n_in, n_out, group, dtype="bf16", zeros=False):
    return {"name": name, "kind": "int4", "rows": rows, "n_in": n_in, "n_out": n_out, "group": group, "dtype": dtype, "zeros": zeros}


def _clip(name, model, d, d_ff, blocks, dtype, norm="2", tensors=0):
    return {"name": name, "kind": "clip", "model": model, "d": d, "d_ff": d_ff, "blocks": blocks, "dtype": dtype, "norm": norm, "tensors": tensors}


def _experts(name, kind, tokens, slots, experts, d, dtype, empty=0.0):
    return {"name": name, "kind": kind, "tokens": tokens, "slots": slots, "experts": experts, "d": d, "dtype": dtype, "empty": empty}


def listed():
    return [
        # one token through the gate_up layer of a block at the benchmark's width: the codes are streamed once
        _int4("int4_1", 1, 2048, 11264, 128),
        # an odd batch of streams through the down layer, finer groups
        _int4("int4_13", 13, 5632, 2048, 64),
        # a small odd batch through widths that fit no tile, in fp16, with zero points and the finest groups
        _int4("int4_odd_77", 77, 1040, 2741, 32, "fp16", True),
        # the benchmark's prompt through the gate_up layer: the largest case
        _int4("int4_4096", 4096, 2048, 11264, 128),
        # the gradients of one base-width router: a few small fp32 tensors, launch latency
        _clip("clip_router", "router", 768, 0, 1, "fp32"),
        # one block at the benchmark's width: two bf16 matrices and its router in fp32
        _clip("clip_block", "block", 2048, 5632, 1, "bf16"),
        # a base-width model of 24 routed blocks
        _clip("clip_model", "block", 768, 2048, 24, "bf16"),
        # hundreds of odd tensors on odd addresses, the largest gradient as the norm
        _clip("clip_ragged", "ragged", 0, 0, 0, "fp16", "inf", 500),
        # one token and its eight experts: launch latency
        _experts("experts_1", "experts_forward", 1, 8, 16, 2048, "bf16"),
        # the benchmark's prompt through 64 experts, eight of them per token
        _experts("experts_4096", "experts_forward", 4096, 8, 64, 2048, "bf16"),
        # a training step at base width, 4 x 4096 tokens, two experts per token
        _experts("experts_train_base", "experts_train", 16384, 2, 16, 768, "bf16"),
        # an odd batch over many experts with empty slots, rows that no vector load fits, in fp16
        _experts("experts_train_odd", "experts_train", 1021, 5, 352, 1999, "fp16", 0.3),
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v // step * step))


def draw(rng):
    kind = rng.choice(["int4", "int4", "clip", "experts_forward", "experts_train"])
    if kind == "int4":
        n_in, n_out = _log_int(rng, 256, 8192, rng.choice([1, 8, 32])), _log_int(rng, 256, 16384, rng.choice([1, 16]))
        rows = max(1, min(_log_int(rng, 1, 16384), int(MAX_INT4_FLOPS / (2.0 * n_in * n_out))))
        c = _int4("", rows, n_in, n_out, rng.choice([32, 64, 128]), rng.choice(["bf16", "fp16"]), rng.random() < 0.3)
    elif kind == "clip":
        model, norm, dtype = rng.choice(["router", "block", "block", "ragged"]), rng.choice(["2", "2", "inf"]), rng.choice(["bf16", "fp16", "fp32"])
        if model == "ragged":
            c = _clip("", model, 0, 0, 0, dtype, norm, _log_int(rng, 2, 1000))
        else:
            d = _log_int(rng, 128, 2048, 16)
            d_ff = _log_int(rng, d, 3 * d, 16) if model == "block" else 0
            c = _clip("", model, d, d_ff, max(1, min(_log_int(rng, 1, 32), MAX_GRADIENTS // (3 * d * d_ff + d * d))), dtype, norm)
    else:
        experts, d = _log_int(rng, 2, 512), _log_int(rng, 64, 4096, rng.choice([1, 8, 8]))
        slots = min(experts, _log_int(rng, 1, 16))
        tokens = max(1, min(_log_int(rng, 1, 16384), MAX_ROUTED_VALUES // (slots * d)))
        c = _experts("", kind, tokens, slots, experts, d, rng.choice(["bf16", "fp16", "fp32"]), rng.choice([0.0, 0.0, 0.3]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- inputs


def _tensors(case):
    """(numel, type) of a clip case's gradients, in the order of a module's parameters."""
    if case["model"] == "ragged":
        return [(1 + (i * 7919 + i * i * 104729) % 20011, case["dtype"]) for i in range(case["tensors"])]
    d, f, t = case["d"], case["d_ff"], case["dtype"]
    keys = max(4, math.ceil(math.sqrt(16)))
    router = [(d * d, "fp32"), (keys * d // 2, "fp32"), (keys * d // 2, "fp32"), (16, "fp32"), (d, "fp32"), (d, "fp32"), (d, "fp32")]
    return (([(2 * f * d, t), (f * d, t), (d, t), (d, t)] if f else []) + router) * case["blocks"]


def _inputs(case, seed):
    """The tensors of a case, made from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    t = DTYPES[case["dtype"]]
    if case["kind"] == "int4":
        n, k = case["n_out"], case["n_in"]
        return {"x": normal(case["rows"], k).to(t), "w": (uniform(n, k) * 2 - 1) / math.sqrt(k)}
    if case["kind"] == "clip":
        sizes, flats, grads = _tensors(case), {}, []
        for name in sorted({s[1] for s in sizes}):
            flat = normal(sum(s[0] for s in sizes if s[1] == name)).to(DTYPES[name])
            flats[name] = [flat, 0]
        for n, name in sizes:
            flat, at = flats[name]
            grads.append(flat[at:at + n])
            flats[name][1] = at + n
        size = torch.exp2(-4.0 - 6.0 * uniform(len(grads)))
        for i, v in enumerate(grads):
            v.mul_(size[i])
        norm = torch.stack([v.float().abs().max() if case["norm"] == "inf" else v.float().norm() for v in grads])
        top = float(norm.max() if case["norm"] == "inf" else norm.norm())
        return {"grads": grads, "flats": {name: f[0] for name, f in flats.items()}, "max_norm": 0.37 * top}
    n, k, e, d = case["tokens"], case["slots"], case["experts"], case["d"]
    score = normal(n, e) + 2.0 * uniform(e)
    top, ids = score.topk(k, dim=1)
    weights = torch.softmax(top, dim=1)
    ids = ids.masked_fill(uniform(n, k) < case["empty"], -1).int()
    s = {"x": normal(n, d).to(t), "ids": ids, "weights": weights, "ys": normal(n * k, d).to(t)}
    if case["kind"] == "experts_train":
        s["dxs"], s["dy"] = normal(n * k, d).to(t), normal(n, d).to(t)
    return s


def _quantise(w, group, zeros, dtype):
    """4-bit codes of a weight [N, K]: words of eight values along K (the rows padded to whole 32), scales [N, ceil(K / group)] of the type and zero points."""
    n, k = w.shape
    groups = -(-k // group)
    p = torch.zeros((n, groups * group), device=w.device)
    p[:, :k] = w
    p = p.view(n, groups, group)
    lo, hi = p.amin(dim=2), p.amax(dim=2)
    s = ((hi - lo) / 15 if zeros else torch.maximum(hi / 7, lo / -8)).to(dtype)
    s = torch.where(s > 0, s, torch.ones_like(s))
    z = (-lo / s.float()).round().clamp(0, 15) if zeros else torch.full_like(lo, 8.0)
    q = ((p / s.float()[:, :, None]).round() + z[:, :, None]).clamp(0, 15).int().view(n, groups * group)
    words = torch.full((n, -(-k // 32) * 32), 8, dtype=torch.int32, device=w.device)
    words[:, :k] = q[:, :k]
    shift = torch.tensor([4 * v for v in NIBBLE], dtype=torch.int64, device=w.device)
    packed = (words.view(n, -1, 8).long() << shift).sum(dim=2)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).int(), s, z.to(torch.uint8) if zeros else None


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "int4":
        s["codes"], s["scales"], s["zeros"] = _quantise(s.pop("w"), case["group"], case["zeros"], DTYPES[case["dtype"]])
        s["group"] = case["group"]
    elif case["kind"] == "clip":
        s["clipped"] = {name: torch.empty_like(f) for name, f in s["flats"].items()}
        at = {name: 0 for name in s["flats"]}
        s["out"] = []
        for (n, name), _ in zip(_tensors(case), s["grads"]):
            s["out"].append(s["clipped"][name][at[name]:at[name] + n])
            at[name] += n
        s["norm"] = math.inf if case["norm"] == "inf" else 2.0
    else:
        s["experts"] = case["experts"]
        if case["kind"] == "experts_train":
            for name in ("x", "weights", "ys"):
                s[name].requires_grad_(True)
    s["kind"] = case["kind"]
    return s


# ---------------------------------------------------------------------------------------------------- one pass


def _run_own(s):
    from mortar_amd import ops
    kind = s["kind"]
    if kind == "int4":
        return ops.linear_int4(s["x"], s["codes"], s["scales"], s["zeros"], group_size=s["group"])
    if kind == "clip":
        _, norm = ops.clip_grads(s["grads"], s["max_norm"], norm_type=s["norm"], out=s["out"])
        return {"norm": norm, **s["clipped"]}
    if kind == "experts_forward":
        with torch.no_grad():
            order = ops.expert_sort(s["ids"], s["experts"])
            xs = ops.expert_dispatch(s["x"], order)
            y = ops.expert_combine(s["ys"], s["weights"], order)
        return order.position, order.token, order.offsets, xs, y
    order = ops.expert_sort(s["ids"], s["experts"])
    xs = ops.expert_dispatch(s["x"], order)
    y = ops.expert_combine(s["ys"], s["weights"], order)
    dx, dys, dw = torch.autograd.grad((xs, y), (s["x"], s["ys"], s["weights"]), (s["dxs"], s["dy"]))
    return order.position, order.token, order.offsets, xs.detach(), y.detach(), dx, dys, dw


def _weight_values(codes, scales, zeros, group, k, t):
    n = codes.shape[0]
    shift = torch.tensor([4 * v for v in NIBBLE], dtype=torch.int32, device=codes.device)
    q = ((codes.unsqueeze(2) >> shift) & 15).view(n, -1)[:, :k].to(t)
    z = zeros.to(t).repeat_interleave(group, 1)[:, :k] if zeros is not None else 8.0
    return (q - z) * scales.to(t).repeat_interleave(group, 1)[:, :k]


def _sorted_order(ids, experts):
    """(position [N, k], token [N k], offsets [E + 1]): the slots stably sorted by expert, the empty ones behind them."""
    k = ids.shape[1]
    key = torch.where((ids >= 0) & (ids < experts), ids, experts).view(-1)
    order = torch.sort(key, stable=True).indices
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=ids.device)
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = counts[:experts].cumsum(0)
    return position.view(-1, k).int(), torch.div(order, k, rounding_mode="floor").int(), offsets


@torch.no_grad()
def _run_plain(s):
    kind = s["kind"]
    if kind == "int4":
        x = s["x"].float()
        return (x @ _weight_values(s["codes"], s["scales"], s["zeros"], s["group"], x.shape[1], torch.float32).t()).to(s["x"].dtype)
    if kind == "clip":
        if math.isinf(s["norm"]):
            norm = torch.stack([g.abs().max().float() for g in s["grads"]]).max()
        else:
            norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]]).sum().sqrt().float()
        c = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        [o.copy_(g.float() * c) for g, o in zip(s["grads"], s["out"])]
        return {"norm": norm, **s["clipped"]}
    position, token, offsets = _sorted_order(s["ids"], s["experts"])
    x, ys, w = s["x"].float(), s["ys"].float(), s["weights"].float()
    t = s["x"].dtype
    full = (s["ids"] >= 0).unsqueeze(2)
    row_full = (torch.arange(ys.shape[0], device=x.device) < offsets[-1]).unsqueeze(1)
    zero = torch.zeros((), device=x.device)
    xs = torch.where(row_full, x[token.long()], zero)
    picked = torch.where(full, ys[position.long()], zero)
    y = (w.unsqueeze(2) * picked).sum(dim=1)
    if kind == "experts_forward":
        return position, token, offsets, xs.to(t), y.to(t)
    dy = s["dy"].float()
    dx = torch.where(full, s["dxs"].float()[position.long()], zero).sum(dim=1)
    dys = torch.empty_like(ys)
    dys[position.view(-1).long()] = torch.where(full, w.unsqueeze(2) * dy.unsqueeze(1), zero).view(-1, ys.shape[1])
    dw = (picked * dy.unsqueeze(1)).sum(dim=2)
    return position, token, offsets, xs.to(t), y.to(t), dx.to(t), dys.to(t), dw


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------- definition


@torch.no_grad()
def exact(case, seed):
    """The definitions in 64 bits."""
    s = _inputs(case, seed)
    if case["kind"] == "int4":
        n, k, group = case["n_out"], case["n_in"], case["group"]
        codes, scales, zeros = _quantise(s["w"], group, case["zeros"], DTYPES[case["dtype"]])
        w = torch.zeros((n, -(-k // 32) * 32), dtype=torch.float64, device=codes.device)
        for j, place in enumerate(NIBBLE):
            w[:, j::8] = (codes >> 4 * place).bitwise_and(15).double()
        for g in range(scales.shape[1]):
            w[:, g * group:(g + 1) * group] -= zeros[:, g:g + 1].double() if zeros is not None else 8.0
            w[:, g * group:(g + 1) * group] *= scales[:, g:g + 1].double()
        return s["x"].double() @ w[:, :k].t()
    if case["kind"] == "clip":
        grads = {name: f.double() for name, f in s["flats"].items()}
        if case["norm"] == "inf":
            norm = max(f.abs().max() for f in grads.values())
        else:
            norm = torch.sqrt(sum(f.dot(f) for f in grads.values()))
        c = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm, **{name: f * c for name, f in grads.items()}}
    n, k, d = case["tokens"], case["slots"], case["d"]
    ids = s["ids"].view(-1)
    full = ids >= 0
    slots = torch.cat([torch.nonzero(ids == e).view(-1) for e in range(case["experts"])] + [torch.nonzero(~full).view(-1)])
    row_of = torch.argsort(slots)
    live = full[slots].unsqueeze(1).double()
    xs = s["x"].double()[slots // k] * live
    rows, w = s["ys"].double()[row_of].view(n, k, d), (s["weights"].double() * full.view(n, k)).unsqueeze(2)
    y = torch.matmul(rows.transpose(1, 2), w).squeeze(2)
    if case["kind"] == "experts_forward":
        return None, None, None, xs, y
    dx = (s["dxs"].double() * live)[row_of].view(n, k, d).sum(dim=1)
    dys = s["dy"].double()[slots // k] * w.view(-1, 1)[slots]
    dw = torch.matmul(rows, s["dy"].double().unsqueeze(2)).squeeze(2) * full.view(n, k)
    return None, None, None, xs, y, dx, dys, dw


def work(case):
    """What no implementation can do without: every input read once, every output written once, the products' multiply-adds."""
    kind, e = case["kind"], 4 if case["dtype"] == "fp32" else 2
    if kind == "int4":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        groups = -(-k // case["group"])
        return {"bytes": e * m * (k + n) + n * k // 2 + n * groups * (3 if case["zeros"] else 2), "flops": 2 * m * n * k}
    if kind == "clip":
        size = {"fp32": 4, "bf16": 2, "fp16": 2}
        sizes = _tensors(case)
        return {"bytes": 2 * sum(n * size[t] for n, t in sizes) + 4, "flops": 3 * sum(n for n, _ in sizes)}
    n, k, d = case["tokens"], case["slots"], case["d"]
    full = n * k * (1.0 - case["empty"])
    index = 4 * (4 * n * k + case["experts"] + 1)               # ids, weights, position, token
    forward = e * d * (n + n * k + full + n)                    # x, xs, ys, y
    if kind == "experts_forward":
        return {"bytes": int(forward + index), "flops": int(2 * full * d)}
    return {"bytes": int(forward + index + e * d * (full + n + n + n * k) + 4 * n * k), "flops": int(7 * full * d)}       # dxs, dx, dy, dys; dw
