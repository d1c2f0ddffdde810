"""Plain forms in 64 bits of the 4-bit layer, gradient clipping and the expert order, and the bounds of their results."""
import torch

from dense_util import U32, rounding

NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)                  # where in its word value j of eight lies


def pack_codes(q):
    """int32 words of the codes q [N, K] (0 .. 15), rows padded to whole 32 values with 8."""
    n, k = q.shape
    p = torch.full((n, -(-k // 32) * 32), 8, dtype=torch.int64, device=q.device)
    p[:, :k] = q
    p = p.view(n, -1, 8)
    w = sum(p[:, :, j] << 4 * NIBBLE[j] for j in range(8))
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def unpack_codes(words, k):
    v = torch.stack([(words.long() >> 4 * NIBBLE[j]) & 15 for j in range(8)], dim=2)
    return v.view(words.shape[0], -1)[:, :k]


def int4_weight(words, scales, zeros, group, k):
    """The weight that the codes stand for, in 64 bits."""
    q = unpack_codes(words, k).double()
    z = zeros.double().repeat_interleave(group, 1)[:, :k] if zeros is not None else 8.0
    return (q - z) * scales.double().repeat_interleave(group, 1)[:, :k]


def quantize_reference(w, group, zero_points):
    """(codes 0 .. 15 [N, K], scales, zeros or None) by the definition, fp32 quotients."""
    n, k = w.shape
    groups = -(-k // group)
    p = torch.zeros((n, groups * group), dtype=torch.float32)
    p[:, :k] = w.float()
    p = p.view(n, groups, group)
    lo, hi = p.amin(2).clamp(max=0), p.amax(2).clamp(min=0)
    s = ((hi - lo) / 15 if zero_points else torch.maximum(hi / 7, lo / -8)).to(w.dtype)
    s = torch.where(s == 0, torch.ones_like(s), s)
    z = (-lo / s.float()).round().clamp(0, 15) if zero_points else torch.full_like(lo, 8.0)
    q = ((p / s.float()[:, :, None]).round() + z[:, :, None]).clamp(0, 15)
    return q.view(n, -1)[:, :k].long(), s, z.to(torch.uint8) if zero_points else None


def int4_bound(x, scales, zeros, group, t, ref):
    """A group's two sums of at most 128 terms |x| 31 and |x| (16 + z) in fp32 (twice half a step per addition, however the matrix cores add), the multiply-adds of the
    groups one behind the other and over 16 waves, and the rounding of the result."""
    m, k = x.shape
    groups = scales.shape[1]
    p = torch.zeros((m, groups * group), dtype=torch.float64, device=x.device)
    p[:, :k] = x.double().abs()
    sx = p.view(m, groups, group).sum(2)
    z = zeros.double() if zeros is not None else torch.full_like(scales, 8.0, dtype=torch.float64)
    size = sx @ (scales.double().abs() * (31 + 16 + z)).t()
    return (2 * 128 + groups + 20) * U32 * size + rounding(t, ref)


def expert_order(ids, n_experts):
    """(position, token, offsets) of the definition."""
    n, k = ids.shape
    key = torch.where((ids >= 0) & (ids < n_experts), ids, n_experts).long().reshape(-1).tolist()
    rows = sorted(range(n * k), key=lambda i: key[i])          # (stable)
    position = torch.empty(n * k, dtype=torch.int32)
    position[torch.tensor(rows, dtype=torch.long)] = torch.arange(n * k, dtype=torch.int32)
    offsets = torch.tensor([sum(v < e for v in key) for e in range(n_experts + 1)] if n_experts < 50 else
                           torch.searchsorted(torch.tensor(sorted(key)), torch.arange(n_experts + 1)).tolist(), dtype=torch.int32)
    return position.view(n, k), torch.tensor(rows, dtype=torch.int32) // k, offsets


def draw_ids(n, k, n_experts, seed, empty=0.3, repeat=False):
    g = torch.Generator().manual_seed(seed)
    if repeat or k > n_experts:
        ids = torch.randint(0, n_experts, (n, k), generator=g)
    else:
        ids = torch.rand((n, n_experts), generator=g).topk(k, dim=1).indices
    return ids.masked_fill(torch.rand((n, k), generator=g) < empty, -1).int()


#: rows, outputs, inputs of 4-bit products: every form of the kernels (a host test looks), odd widths, ends inside a word, a group, a chunk, a tile
INT4_SIZES = [(1, 1, 1), (1, 16, 32), (1, 17, 40), (2, 24, 128), (3, 130, 257), (5, 264, 2120), (2, 8200, 4000), (13, 264, 1040), (16, 2048, 5632), (17, 136, 400), (31, 33, 264),
              (32, 256, 1999), (33, 256, 144), (64, 520, 1040), (65, 9, 72), (96, 1031, 264), (96, 1031, 1040), (129, 264, 400), (130, 127, 2736), (200, 1031, 1040), (300, 135, 272),
              (520, 1031, 264), (5000, 130, 72), (2100, 2056, 392), (4200, 264, 264), (6000, 517, 136), (300, 2055, 8200), (4200, 131, 4104),
              (4200, 136, 2056), (1000, 1031, 4104), (200, 4103, 4104), (13, 8200, 264), (33, 8200, 136), (17, 8200, 1040), (70, 4103, 1999), (2000, 520, 6152),
              (5, 264, 2560), (13, 264, 5632), (9, 40, 7680), (7, 8200, 4096), (3, 130, 1024)]
