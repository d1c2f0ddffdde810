"""CPU tests of the 4-bit layer, clipping and the expert order: what is refused before anything is launched, and the 64-bit forms that the GPU tests compare with."""
import ctypes as C
import math

import pytest
import torch

from mortar_amd import _lib, ops
from operators_util import INT4_SIZES, draw_ids, expert_order, int4_weight, pack_codes, quantize_reference, unpack_codes

A = 1 << 20                                   # an aligned address that is never read: every call here is refused


def _refused(rc, code=-1):
    assert rc == code and _lib.lib().mortar_last_error()


def test_int4_linear_refuses():
    f = _lib.lib().mortar_int4_linear
    base = dict(x=A, M=1, K=64, ldx=64, type=0, c=A, ldc=8, N=16, group=32, s=A, s_type=0, s_n=1, s_g=16, z=None, z_n=0, z_g=0, y=A, ldy=16, ws=None, st=None)
    call = lambda **k: f(*{**base, **k}.values())
    for bad in (dict(M=-1), dict(K=0), dict(N=0), dict(type=2), dict(s_type=1), dict(s_type=3), dict(group=16), dict(group=0), dict(group=256), dict(x=None), dict(x=A + 2),
                dict(K=60), dict(ldx=60), dict(M=2, ldx=56), dict(c=None), dict(c=A + 4), dict(ldc=4), dict(ldc=9), dict(s=None), dict(y=None), dict(y=A + 1), dict(ldy=15),
                dict(s_n=-1), dict(s_g=-1), dict(z_n=-1), dict(z_g=-1), dict(M=5000, ldy=16)):
        _refused(call(**bad))
    _refused(call(ldc=1 << 22), -4)
    _refused(call(ldx=1 << 23), -4)
    _refused(call(N=1 << 24, ldy=1 << 24), -4)
    assert call(M=0, x=None, c=None, s=None, y=None) == 0
    ws = _lib.lib().mortar_int4_workspace_bytes
    assert ws(1, 16, 64, 32) == 0 and ws(0, 16, 64, 32) == 0 and ws(5000, 16, 64, 32) == 4 * 2 * (5120 + 2 * 128)


def _form(M, N, K, group):
    v = [C.c_int32() for _ in range(4)]
    assert _lib.lib().mortar_int4_form_host(M, N, K, group, *[C.byref(i) for i in v]) == 0
    return tuple(i.value for i in v)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_sizes_reach_every_form(group):
    """Rows of x through LDS, straight from memory, and tiles of one and of several ranges of K."""
    few = [(16, 16, -8), (16, 16, -16), (32, 16, -16), (64, 32, 8)] + [(16 * f, 16, w) for f in (1, 2, 4) for w in (8, 16)]
    forms = {_form(*s, group) for s in INT4_SIZES}
    assert {f[:3] for f in forms if f[3] == 1} == {*few, (64, 64, 4), (128, 128, 4)}
    assert {f[:2] for f in forms if f[3] > 1} == {(64, 64), (128, 128)}
    f = _lib.lib().mortar_int4_form_host
    _refused(f(0, 16, 64, group, A, A, A, A))
    _refused(f(1, 16, 64, 16, A, A, A, A))
    _refused(f(1, 16, 64, group, A, A, A, None))


def test_int4_rows_refuses():
    f = _lib.lib().mortar_int4_rows
    for bad in ((A, -1, 8, 8, 1, A), (A, 1, 0, 8, 1, A), (None, 1, 8, 8, 1, A), (A, 1, 8, 8, 1, None), (A + 1, 1, 8, 8, 1, A), (A, 1, 8, 8, 1, A + 8)):
        _refused(f(*bad, None))
    _refused(f(A, 1 << 32, 8, 8, 1, A, None), -4)
    assert f(None, 0, 8, 8, 1, None, None) == 0


def test_int4_quantize_refuses():
    f = _lib.lib().mortar_int4_quantize
    base = dict(w=A, N=16, K=64, ldw=64, type=0, group=32, c=A, ldc=8, s=A, s_type=0, s_n=1, s_g=16, z=None, z_n=0, z_g=0, st=None)
    call = lambda **k: f(*{**base, **k}.values())
    for bad in (dict(N=0), dict(K=0), dict(type=3), dict(s_type=-1), dict(group=48), dict(c=None), dict(c=A + 8), dict(ldc=4), dict(w=None), dict(s=None), dict(ldw=63)):
        _refused(call(**bad))
    _refused(call(N=(1 << 31) - 1, K=1 << 20, ldw=1 << 20, ldc=1 << 17), -4)


def _grads(*entries):
    return (_lib.GradStruct * max(1, len(entries)))(*[_lib.GradStruct(*e) for e in entries]), len(entries)


def test_gradients_refuse():
    L = _lib.lib()
    good = (A, A, 10, 0, 0)
    for bad in ((A, A, -1, 0, 0), (A, A, 10, 3, 3), (None, A, 10, 0, 0), (A + 1, A, 10, 0, 0), (A + 2, A, 10, 2, 2)):
        g, n = _grads(good, bad)
        _refused(L.mortar_grad_norm(g, n, 0, A, A, None))
        _refused(L.mortar_grad_workspace_bytes(g, n))
    for bad in ((A, A, 10, 0, 1), (A, A, 10, 2, 0), (A, None, 10, 0, 0), (A, A + 1, 10, 0, 0), (A, A + 2, 10, 0, 2), (A, A, 10, 0, 7)):
        g, n = _grads(good, bad)
        _refused(L.mortar_grad_clip(g, n, 0, 1.0, A, A, None))
    g, n = _grads(good)
    _refused(L.mortar_grad_norm(g, -1, 0, A, A, None))
    _refused(L.mortar_grad_norm(None, 1, 0, A, A, None))
    _refused(L.mortar_grad_norm(g, n, 0, None, A, None))
    _refused(L.mortar_grad_norm(g, n, 0, A, None, None))
    _refused(L.mortar_grad_clip(g, n, 0, -1.0, A, A, None))
    _refused(L.mortar_grad_clip(g, n, 0, math.nan, A, A, None))
    huge, n = _grads((A, A, 1 << 40, 0, 0))
    _refused(L.mortar_grad_norm(huge, n, 0, A, A, None), -4)
    g, n = _grads(*[(A, A, 1, 0, 0)] * 300, *[(None, None, 0, 0, 0)] * 7)
    assert L.mortar_grad_workspace_bytes(g, n) == 8 * 301
    g, n = _grads((A, A, 1 << 35, 0, 0))
    assert L.mortar_grad_workspace_bytes(g, n) == 8 * 1025


def test_experts_refuse():
    L = _lib.lib()
    sort = lambda **k: L.mortar_expert_sort(*{**dict(ids=A, i64=0, N=4, k=2, e=8, p=A, t=A, o=A, ws=None, st=None), **k}.values())
    for bad in (dict(N=-1), dict(k=0), dict(e=0), dict(ids=None), dict(p=None), dict(t=None), dict(o=None), dict(N=5000)):
        _refused(sort(**bad))
    _refused(sort(e=1025), -4)
    _refused(sort(N=1 << 25), -4)
    _refused(sort(N=1 << 40), -4)
    assert L.mortar_expert_sort_workspace_bytes(4096, 8) == 0 and L.mortar_expert_sort_workspace_bytes(1 << 20, 8) > 0
    disp = lambda **k: L.mortar_expert_dispatch(*{**dict(x=A, N=4, d=8, ld=8, t=0, k=2, p=A, f=A, xs=A, st=None), **k}.values())
    for bad in (dict(N=-1), dict(d=0), dict(k=0), dict(t=5), dict(x=None), dict(x=A + 1), dict(t=2, x=A + 2), dict(p=None), dict(f=None), dict(xs=None), dict(xs=A + 1), dict(p=A + 2)):
        _refused(disp(**bad))
    comb = lambda **k: L.mortar_expert_combine(*{**dict(ys=A, N=4, d=8, t=0, k=2, p=A, f=A, w=A, wt=2, y=A, st=None), **k}.values())
    for bad in (dict(N=-1), dict(d=0), dict(k=0), dict(t=5), dict(ys=None), dict(y=None), dict(y=A + 1), dict(p=None), dict(f=None), dict(wt=4), dict(w=A + 2)):
        _refused(comb(**bad))
    bwd = lambda **k: L.mortar_expert_combine_bwd(*{**dict(dy=A, ld=8, ys=A, N=4, d=8, t=0, k=2, p=A, f=A, w=A, wt=2, dys=A, dw=A, st=None), **k}.values())
    for bad in (dict(N=-1), dict(d=0), dict(t=5), dict(dy=None), dict(ys=None), dict(p=None), dict(f=None), dict(wt=4), dict(w=A + 2), dict(dys=A + 1), dict(dw=A + 1)):
        _refused(bwd(**bad))
    assert disp(N=0) == 0 and comb(N=0) == 0 and bwd(N=0) == 0 and bwd(dys=None, dw=None) == 0


def test_tensors_on_the_cpu_are_refused():
    x, i = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((2, 1), dtype=torch.int32)
    order = ops.ExpertOrder(i, i.view(-1), torch.zeros(3, dtype=torch.int32))
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    for call in (lambda: ops.quantize_int4_weight(x), lambda: ops.linear_int4(x, torch.zeros((8, 8), dtype=torch.int32), x), lambda: ops.grad_norm([x]),
                 lambda: ops.clip_grads([x], 1.0), lambda: ops.clip_grad_norm_(p, 1.0), lambda: ops.expert_sort(i, 2), lambda: ops.expert_dispatch(x, order),
                 lambda: ops.expert_combine(x, None, order)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_arguments_of_the_wrong_kind():
    with pytest.raises(ValueError, match="norm_type"):
        ops.grad_norm([], 3)
    with pytest.raises(ValueError, match="norm_type"):
        ops.clip_grad_norm_([], 1.0, norm_type=1)
    with pytest.raises(TypeError, match="tensor"):
        ops.grad_norm([3])
    with pytest.raises(TypeError):
        ops.grad_norm(3)
    with pytest.raises(TypeError, match="tensor"):
        ops.expert_sort([[0]], 2)
    with pytest.raises(ValueError, match="max_norm"):
        ops.clip_grads([], -1.0)


def test_no_gradients_at_all():
    """As torch's clipping: a norm of 0, nothing to do."""
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(ops.grad_norm([])) == 0.0 and ops.clip_grads([], 1.0)[0] == []
    assert float(ops.clip_grad_norm_([p], 1.0)) == 0.0 and float(ops.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)) == 0.0


def test_codes_round_trip():
    q = torch.randint(0, 16, (5, 77), generator=torch.Generator().manual_seed(0))
    words = pack_codes(q)
    assert words.shape == (5, 12) and torch.equal(unpack_codes(words, 77), q) and bool((unpack_codes(words, 96)[:, 77:] == 8).all())


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_reference_is_near(zeros):
    """A value is off by half a step, and by what clamping at the end of the range and the rounding of the scale to bf16 take: one step in all."""
    w = torch.randn((7, 200), generator=torch.Generator().manual_seed(1)).bfloat16()
    q, s, z = quantize_reference(w, 64, zeros)
    v = int4_weight(pack_codes(q), s, z, 64, 200)
    assert bool(((v - w.double()).abs() <= s.double().repeat_interleave(64, 1)[:, :200]).all())


def test_order_reference():
    ids = draw_ids(40, 3, 6, 2)
    position, token, offsets = expert_order(ids, 6)
    assert sorted(position.view(-1).tolist()) == list(range(120))
    flat = ids.view(-1)
    for i in range(120):
        r, e = int(position.view(-1)[i]), int(flat[i])
        assert int(token[r]) == i // 3
        assert offsets[e] <= r < offsets[e + 1] if e >= 0 else r >= offsets[6]
