"""CPU tests of the layers that are not carved: hooks, 8-bit state dictionaries, masks and casts of packed layers."""
import copy

import pytest
import torch

from mortar_amd.block_sparse import CMSBlockLinear
from mortar_amd.mlp import call_is_forward

K, N = 160, 272


@pytest.mark.parametrize("register", [
    lambda m, f: m.register_full_backward_hook(f), lambda m, f: m.register_full_backward_pre_hook(f), lambda m, f: m.register_forward_hook(f),
    lambda m, f: m.register_forward_pre_hook(f), lambda m, f: torch.nn.modules.module.register_module_full_backward_hook(f),
    lambda m, f: torch.nn.modules.module.register_module_full_backward_pre_hook(f), lambda m, f: torch.nn.modules.module.register_module_forward_hook(f),
    lambda m, f: torch.nn.modules.module.register_module_forward_pre_hook(f)],
    ids=["backward", "backward_pre", "forward", "forward_pre", "global_backward", "global_backward_pre", "global_forward", "global_forward_pre"])
def test_a_layer_with_hooks_is_called(register):
    lin = CMSBlockLinear(32, 32)
    assert call_is_forward(lin, CMSBlockLinear.forward)
    handle = register(lin, lambda *a: None)
    try:
        assert not call_is_forward(lin, CMSBlockLinear.forward)
    finally:
        handle.remove()
    assert call_is_forward(lin, CMSBlockLinear.forward)
