"""What the C entries of the 4-bit layer, clipping and the expert rows refuse at their edges, before anything is launched."""
import pytest

from mortar_amd import _lib

A = 1 << 20                                   # an aligned address that is never read: every call here is refused


def _refused(rc, code=-1):
    assert rc == code and _lib.lib().mortar_last_error()


@pytest.mark.parametrize("used", [65, 56, 0, -1])
def test_int4_part_refuses(used):
    """Fewer than eight of the K values may be padding."""
    f = _lib.lib().mortar_int4_linear_part
    base = dict(x=A, M=1, K=64, used=used, ldx=64, type=0, c=A, ldc=8, N=16, group=32, s=A, s_type=0, s_n=1, s_g=16, z=None, z_n=0, z_g=0, y=A, ldy=16, ws=None, st=None)
    _refused(f(*base.values()))
    assert f(*{**base, "used": 57, "M": 0}.values()) == 0


@pytest.mark.parametrize("N,k", [((1 << 26) - 3, 1), ((1 << 26) - 1, 1), (33554431, 2), (22369621, 3), (1 << 26, 1), (1, (1 << 26) - 1)])
def test_more_slots_than_a_launch_has_waves(N, k):
    """A wave per slot, four to a workgroup of 256, and fewer than 2^32 threads: 2^26 - 4 slots at most."""
    L = _lib.lib()
    assert N * k > (1 << 26) - 4
    _refused(L.mortar_expert_sort(A, 0, N, k, 8, A, A, A, A, None), -4)
    _refused(L.mortar_expert_dispatch(A, N, 8, 8, 0, k, A, A, A, None), -4)
    _refused(L.mortar_expert_dispatch_rows(A, N, 8, 8, 0, k, A, A, A, A, None), -4)
    _refused(L.mortar_expert_combine(A, N, 8, 0, k, A, A, A, 2, A, None), -4)
    _refused(L.mortar_expert_combine_bwd(A, 8, A, N, 8, 0, k, A, A, A, 2, A, A, None), -4)
    _refused(L.mortar_expert_combine_bwd_rows(A, 8, A, N, 8, 0, k, A, A, A, A, 2, A, A, None), -4)
