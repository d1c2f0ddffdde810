"""Calls at the edges of the dense operators: what hangs on the layers of a fused MLP, calls that only torch's layers cover, rows far apart, values
at the ends of the range, gradients and scales in unusual forms."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from dense_util import assert_within, normals, rounding
from mortar_amd import _lib, ops
from mortar_amd.mlp import _SwiGLUMortar

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _mlp(dev, d=64, f=96, t=BF16):
    torch.manual_seed(0)
    mlp = _SwiGLUMortar(d, f).to(dev).to(t)
    mlp.dense_fused = True
    return mlp


# ---- the MLP's modules


@pytest.mark.parametrize("kind", ["backward", "backward_pre", "global_backward", "global_backward_pre"])
@pytest.mark.parametrize("where", ["gate_up", "gate_up._cms", "down", "down._cms"])
def test_backward_hooks_of_the_layers_run(dev, where, kind):
    mlp = _mlp(dev)
    m, seen = mlp.get_submodule(where), []
    see = lambda mod, *a: seen.append(mod) if mod is m else None
    if kind == "backward":
        handle = m.register_full_backward_hook(see)
    elif kind == "backward_pre":
        handle = m.register_full_backward_pre_hook(see)
    elif kind == "global_backward":
        handle = torch.nn.modules.module.register_module_full_backward_hook(see)
    else:
        handle = torch.nn.modules.module.register_module_full_backward_pre_hook(see)
    try:
        x = normals((5, 64), 1, BF16, dev).requires_grad_(True)
        mlp(x).sum().backward()
    finally:
        handle.remove()
    assert seen == [m]
