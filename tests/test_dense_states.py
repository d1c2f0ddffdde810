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


def _codes(n=N, k=K, seed=0):
    """The two buffers of a packed layer, as pack_dense_fp8 makes them."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randn((n, k), generator=g).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, torch.rand((-(-n // 128), -(-k // 128)), generator=g) / 7


def _packed(seed=0, bias=False):
    lin = CMSBlockLinear(K, N, bias=bias)
    state = {"dense_fp8": _codes(seed=seed)[0], "dense_fp8_scale": _codes(seed=seed)[1]}
    if bias:
        state["bias"] = torch.arange(N, dtype=torch.float32)
    lin.load_state_dict(state)
    return lin, state


def _holds(lin, state):
    return all(torch.equal(lin.state_dict()[k], v) and lin.state_dict()[k].dtype == v.dtype for k, v in state.items()) and lin.state_dict().keys() == state.keys()


def test_packed_state_loads():
    for bias in (False, True):
        lin, state = _packed(bias=bias)
        assert "weight" not in lin._parameters and _holds(lin, state)
        lin.load_state_dict({**state, "dense_fp8_scale": state["dense_fp8_scale"] * 2})            # and once more, into a packed layer
        assert torch.equal(lin.dense_fp8_scale, state["dense_fp8_scale"] * 2)


@pytest.mark.parametrize("strict", [True, False])
@pytest.mark.parametrize("into_packed", [False, True])
@pytest.mark.parametrize("n,k,rows,cols", [(N + 16, K, 3, 2), (N, K + 16, 3, 2), (N, K, 4, 2), (N, K, 3, 3), (16, K, 1, 2)])
def test_packed_state_of_another_size_is_an_error(n, k, rows, cols, into_packed, strict):
    """As for every other parameter, in strict and other loads: the layer keeps its features."""
    lin = _packed(seed=3)[0] if into_packed else CMSBlockLinear(K, N, bias=False)
    before = {k: v.clone() for k, v in lin.state_dict().items()}
    with pytest.raises(RuntimeError, match="size mismatch"):
        lin.load_state_dict({"dense_fp8": _codes(n, k)[0], "dense_fp8_scale": torch.ones(rows, cols)}, strict=strict)
    assert _holds(lin, before)


@pytest.mark.parametrize("missing", ["dense_fp8", "dense_fp8_scale"])
def test_half_a_packed_state_leaves_the_layer_alone(missing):
    """Codes without scales (or the other way round) are missing keys, reported as such; the layer still has its weight."""
    lin = CMSBlockLinear(K, N, bias=False)
    weight = lin.weight.detach().clone()
    _, state = _packed()
    del state[missing]
    with pytest.raises(RuntimeError, match="[Mm]issing key"):
        lin.load_state_dict(state)
    assert torch.equal(lin.weight, weight) and "dense_fp8" not in lin._buffers and "dense_fp8_scale" not in lin._buffers
    result = lin.load_state_dict(state, strict=False)
    assert result.missing_keys == ["weight"] and torch.equal(lin.weight, weight)


def test_a_carved_state_loads_into_a_packed_layer():
    torch.manual_seed(0)
    carved = CMSBlockLinear(K, N, bias=False)
    carved.carve()
    lin, _ = _packed()
    lin.load_state_dict(carved.state_dict())
    assert lin._mortar and not lin._dense_mode and "dense_fp8" not in lin._buffers and "dense_fp8_scale" not in lin._buffers and "weight" not in lin._parameters
    assert _holds(lin, carved.state_dict())


def test_a_mask_on_a_packed_layer_is_refused():
    lin, state = _packed()
    with pytest.raises(AssertionError, match="8-bit codes"):
        lin.set_block_mask(torch.ones(N // 16, K // 16, dtype=torch.bool))
    assert lin._prune_mask is None and _holds(lin, state)


def test_codes_and_scales_of_other_types_are_an_error():
    """They are no numbers that a copy may round: scales in 16 bits, codes as floats."""
    codes, scale = _codes()
    for into in (CMSBlockLinear(K, N, bias=False), _packed(seed=3)[0]):
        for state in ({"dense_fp8": codes, "dense_fp8_scale": scale.bfloat16()}, {"dense_fp8": codes.float(), "dense_fp8_scale": scale}):
            with pytest.raises(RuntimeError, match="must be"):
                into.load_state_dict(state)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_scales_are_whole_again_behind_a_cast(t):
    """A module that was cast to 16 bits and back holds the scales that it was packed with, not rounded ones."""
    lin, state = _packed(bias=True)
    assert not torch.equal(state["dense_fp8_scale"].to(t).float(), state["dense_fp8_scale"])
    cast = lin.to(t)
    assert cast.dense_fp8.dtype == torch.uint8 and torch.equal(cast.dense_fp8, state["dense_fp8"])
    for back in (copy.deepcopy(cast).float(), copy.deepcopy(cast).to(torch.float16).bfloat16().float(), copy.deepcopy(cast).double().float(), cast.float()):
        assert back.dense_fp8_scale.dtype == torch.float32 and torch.equal(back.dense_fp8_scale, state["dense_fp8_scale"])
    cast, new = lin.to(t), _codes(seed=9)
    assert _holds(cast, {**state, "bias": state["bias"].to(t)})                       # a checkpoint of it is whole, too
    with pytest.raises(RuntimeError, match="float32"):
        cast.load_state_dict({"dense_fp8": new[0], "dense_fp8_scale": new[1], "bias": state["bias"]})
    lin, state = _packed(seed=2)
    assert torch.equal(lin.double().dense_fp8_scale.float(), state["dense_fp8_scale"])


def test_scales_that_are_set_anew_behind_a_cast():
    """The layer's own buffer counts, whatever was kept through a cast."""
    lin, state = _packed()
    new = state["dense_fp8_scale"] * 2
    lin.bfloat16().dense_fp8_scale = new.clone()
    assert torch.equal(lin.state_dict()["dense_fp8_scale"], new) and torch.equal(copy.deepcopy(lin).float().dense_fp8_scale, new)
    lin.load_state_dict(state)
    assert _holds(lin, state) and torch.equal(lin.bfloat16().float().dense_fp8_scale, state["dense_fp8_scale"])
