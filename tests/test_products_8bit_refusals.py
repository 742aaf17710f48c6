"""Products in 8-bit integers on the host: what the entry points refuse before anything is launched."""
import pytest
import torch

from fieldrun_b200.csrc import ops


@pytest.mark.parametrize("place", [1, 4, 8, 255])
def test_scratch_off_16_bytes_is_refused_before_any_kernel_writes_to_it(place):
    lib, room = ops.library("products8"), 1 << 40
    calls = {
        "linear": lambda: lib.frb_linear_8bit(None, 0, 9, 100, None, None, 33, None, 0, 0, place, room, None, None),
        "gated block": lambda: lib.frb_gated_8bit(None, 0, 3, 100, None, None, 40, None, None, 0, 0.0, None, 0, 0, place, room, None, None),
        "experts": lambda: lib.frb_expert_rows_8bit(None, 0, 3, 100, 1, None, None, None, None, None, 5, 8, None, None, 5, 40, None, None, 0.0, None, place, room, None,
                                                    None),
        "experts ": lambda: lib.frb_experts_8bit(None, 0, 3, 100, 2, None, None, None, None, 5, 40, None, None, 0.0, 8, None, 0, place, room, None, None),
    }
    for what, call in calls.items():
        assert call() == -1, what
        assert lib.frb_last_error().decode() == f"{what.strip()} in 8 bits: the scratch starts on 16 bytes"


def weight(experts, parts, features, inner):
    shape = ops.weight_8bit_shape(experts, parts, features, inner)
    return torch.zeros(shape, dtype=torch.int8), torch.zeros(shape[:3])


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def blocks(tokens):
    """Calls of the gated operators for so many tokens, each with options of its own."""
    x, w_in, w_down = torch.zeros(tokens, 100), weight(5, 2, 40, 100), weight(5, 1, 100, 40)
    lists = (ints(6), ints(6), ints(1), ints(6))
    return {
        "gated_8bit": lambda **more: ops.gated_8bit(x, *weight(1, 2, 40, 100), *weight(1, 1, 100, 40), x.clone(), width=40, **more),
        "expert_rows_8bit": lambda **more: ops.expert_rows_8bit(x, None, lists, 6, 8, *w_in, *w_down, x.clone(), width=40, **more),
        "experts_8bit": lambda **more: ops.experts_8bit(x, ints(tokens, 2), torch.zeros(tokens, 2), *w_in, *w_down, x.clone(), width=40, **more)}


@pytest.mark.parametrize("limit", [float("nan"), -1.0, -float("inf")])
def test_a_gate_limit_that_is_none_is_refused(limit):
    for name, call in blocks(3).items():
        with pytest.raises(ops.KernelError, match=f"{name}: .*a gate limit of {limit}"):
            call(gate_limit=limit)


@pytest.mark.parametrize("tokens", [0, 3])
def test_kernels_counted(tokens, monkeypatch):
    """What a call of no tokens launches is nothing; three tokens' linear layer is one kernel, their gated block two, their experts six."""
    monkeypatch.setattr(ops, "_addresses", lambda *tensors: [0] * len(tensors))
    monkeypatch.setattr(ops, "_status_at", lambda device: 0)
    monkeypatch.setattr(ops, "_call", lambda name, *args: ops.count_launches(ops._KERNELS_PER_CALL[name]))
    calls = blocks(tokens)
    calls["linear_8bit"] = lambda: ops.linear_8bit(torch.zeros(tokens, 100), *weight(1, 1, 40, 100), torch.zeros(tokens, 40))
    for name, kernels in {"linear_8bit": 1, "gated_8bit": 2, "experts_8bit": 6}.items():
        before = ops.launches()
        calls[name]()
        assert ops.launches() - before == (kernels if tokens else 0), name


def test_a_weights_places_come_together():
    codes, scales = weight(1, 1, 40, 100)
    matrix = torch.zeros(40, 100)
    for more in (dict(codes=codes), dict(scales=scales)):
        with pytest.raises(ops.KernelError, match="codes and scales come together"):
            ops.weight_8bit(matrix, **more)
    with pytest.raises(ops.KernelError, match="weights of shapes \\[\\]: one matrix"):
        ops.weight_8bit()
    with pytest.raises(ops.KernelError, match="a CPU tensor was given"):
        ops.weight_8bit(matrix, codes=codes, scales=scales)
