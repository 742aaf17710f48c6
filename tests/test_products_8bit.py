"""Products in 8-bit integers on the host: what their calls refuse."""
import pytest
import torch

from fieldrun_b200.csrc import ops
from plain_products_8bit import up

HOST = "a CPU tensor was given"


def refuses(call, args, options, at, value, match):
    """The call with one of its arguments (a place or a name) put in another's place."""
    args, options = list(args), dict(options)
    if isinstance(at, int):
        args[at] = value
    else:
        options[at] = value
    with pytest.raises(ops.KernelError, match=match):
        call(*args, **options)


def weight(experts, parts, features, inner):
    shape = ops.weight_8bit_shape(experts, parts, features, inner)
    return torch.zeros(shape, dtype=torch.int8), torch.zeros(shape[:3])


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_layout():
    assert ops.weight_8bit_shape(3, 2, 17, 129) == (3, 2, 32, 256) and ops.weight_8bit_shape(1, 1, 16, 128) == (1, 1, 16, 128)


def test_what_rows_refuse():
    args = (torch.zeros(3, 100), torch.zeros(3, 128, dtype=torch.int8), torch.zeros(3))
    with pytest.raises(ops.KernelError, match=HOST):
        ops.rows_8bit(*args)
    for at, value, match in [(0, torch.zeros(300), "rows of shape"), (0, torch.zeros(3, 0), "rows of shape"), (0, torch.zeros(1, 131073), "1 to 131072"),
                             (1, torch.zeros(3, 100, dtype=torch.int8), "codes of shape"), (1, torch.zeros(3, 128), "codes of rows must be"),
                             (2, torch.zeros(3).double(), "scales of rows must be"), (2, torch.zeros(4), "with scales of")]:
        refuses(ops.rows_8bit, args, {}, at, value, match)
    for parts, match in [((torch.zeros(3, 4), torch.zeros(3, 5)), "of one shape"), ((torch.zeros(3, 4),) * 3, "of one shape"), ((torch.zeros(12),), "one matrix"),
                         ((torch.zeros(0, 12),), "one matrix")]:
        with pytest.raises(ops.KernelError, match=match):
            ops.weight_8bit(*parts)
    with pytest.raises(ops.KernelError, match="not \\[1, 1, 16, 128\\]"):
        ops.weight_8bit(torch.zeros(3, 4), codes=torch.zeros(1, 1, 16, 4, dtype=torch.int8), scales=torch.zeros(1, 1, 16))


def test_what_a_linear_layer_refuses():
    w, s = weight(1, 1, 33, 100)
    args = (torch.zeros(3, 100), w, s, torch.zeros(3, 33))
    with pytest.raises(ops.KernelError, match=HOST):
        ops.linear_8bit(*args)
    for at, value, match in [
            (0, torch.zeros(3, 300), "codes of shape"), (0, torch.zeros(2, 100), "with results of"), (0, torch.zeros(300), "rows of shape"),
            (1, w.float(), "codes are int8"), (1, w[0, 0], "codes of shape"), (1, w[:, :, :33], "codes of shape"), (1, w[..., :100], "codes of shape"),
            (1, torch.zeros(2, 1, 48, 128, dtype=torch.int8), "codes of shape"), (2, s.double(), "scales float32"), (2, s[..., :33], "with scales of"),
            (3, torch.zeros(3, 60), "codes of shape"), (3, torch.zeros(4, 33), "with results of"), (3, torch.zeros(3, 0), "with results of"),
            ("scratch", torch.zeros(4096), "as scratch")]:
        refuses(ops.linear_8bit, args, {}, at, value, match)
    refuses(ops.linear_8bit, (torch.zeros(9, 100), w, s, torch.zeros(9, 33)), {}, "scratch", torch.zeros(64, dtype=torch.uint8), "are needed")
    assert ops.linear_8bit_scratch(3, 100) == 0 and ops.linear_8bit_scratch(9, 100) == 9 * 128 + 128 + 256      # runs of 256 bytes


def test_what_a_gated_block_refuses():
    args = (torch.zeros(3, 100), *weight(1, 2, 40, 100), *weight(1, 1, 100, 40), torch.zeros(3, 100))
    options = dict(width=40)
    with pytest.raises(ops.KernelError, match=HOST):
        ops.gated_8bit(*args, **options)
    for at, value, match in [
            (0, torch.zeros(3, 99), "with results of"), (1, weight(1, 1, 40, 100)[0], "gate and up: codes of shape"), (2, weight(1, 2, 60, 100)[1], "gate and up: "),
            (3, weight(1, 1, 40, 100)[0], "down: codes of shape"), (4, torch.zeros(1, 1, 100), "down: "), (5, torch.zeros(3, 40), "with results of"),
            ("width", 0, "a width of 0"), ("width", 60, "gate and up: codes"), ("activation", "relu", "activation 'relu'"), ("gate_limit", -1.0, "a gate limit of -1.0")]:
        refuses(ops.gated_8bit, args, options, at, value, match)
    refuses(ops.gated_8bit, args, dict(width=40, gate_limit=7.0), "activation", "gelu_tanh", "gate limit of 7.0")


def test_what_experts_refuse():
    args = (torch.zeros(3, 100), ints(3, 2), torch.zeros(3, 2), *weight(5, 2, 40, 100), *weight(5, 1, 100, 40), torch.zeros(3, 100))
    options = dict(width=40)
    with pytest.raises(ops.KernelError, match=HOST):
        ops.experts_8bit(*args, **options)
    for at, value, match in [
            (0, torch.zeros(4, 100), "with results of"), (1, ints(6), "ids of shape"), (1, ints(3, 2).long(), "must be torch.int32"), (1, ints(3, 3), "for 3 tokens"),
            (2, torch.zeros(3, 2).double(), "the experts' weights must be"), (2, torch.zeros(2, 2), "and weights of"), (3, weight(5, 1, 40, 100)[0], "gate and up"),
            (5, weight(4, 1, 100, 40)[0], "down: codes"), (7, torch.zeros(3, 40), "with results of"), ("width", 131073, "a width of"), ("gate_limit", -0.5, "gate limit")]:
        refuses(ops.experts_8bit, args, options, at, value, match)
    refuses(ops.experts_8bit, (args[0], ints(3, 129), torch.zeros(3, 129), *args[3:]), options, "width", 40, "1 to 128 experts")


def test_what_expert_rows_refuse():
    lists = (ints(6), ints(6), ints(1), ints(6))
    args = (torch.zeros(3, 100), ints(6), lists, 6, 8, *weight(5, 2, 40, 100), *weight(5, 1, 100, 40), torch.zeros(6, 100))
    options = dict(width=40)
    with pytest.raises(ops.KernelError, match=HOST):
        ops.expert_rows_8bit(*args, **options)
    for at, value, match in [
            (0, torch.zeros(4, 100), "rows of experts"), (1, ints(6).long(), "must be torch.int32"), (1, ints(7), "7 rows of experts"),
            (2, (*lists[:3], ints(5)), "lists of"), (2, (lists[0].float(), *lists[1:]), "must be torch.int32"), (3, 0, "0 tiles"), (3, 7, "lists of"), (4, 24, "tiles of 24 rows"),
            (9, torch.zeros(6, 100).double(), "expert outputs must be"), (9, torch.zeros(5, 100), "with 6 rows"), ("width", 57, "gate and up: codes")]:
        refuses(ops.expert_rows_8bit, args, options, at, value, match)


def test_entry_points_refuse_sizes_by_a_message():
    # the C entry points' own checks, which come before anything is launched
    lib = ops.library("products8")
    assert lib.frb_linear_8bit(None, 0, 9, 100, None, None, 33, None, 0, 0, None, ops.linear_8bit_scratch(9, 100) - 1, None, None) == -1
    assert b"are needed" in lib.frb_last_error()
    assert lib.frb_linear_8bit(None, 0, 3, 131073, None, None, 33, None, 0, 0, None, 1 << 40, None, None) == -1
    assert b"131073 entries" in lib.frb_last_error()
    assert lib.frb_gated_8bit(None, 0, 3, 100, None, None, 40, None, None, 0, 0.0, None, 0, 0, None, ops.gated_8bit_scratch(3, 100, 40) - 1, None, None) == -1
    assert b"are needed" in lib.frb_last_error()
    assert lib.frb_gated_8bit(None, 0, 3, 100, None, None, 40, None, None, 2, 0.0, None, 0, 0, None, 1 << 40, None, None) == -1
    assert b"activation 2" in lib.frb_last_error()
    assert lib.frb_experts_8bit(None, 0, 1 << 24, 100, 128, None, None, None, None, 5, 40, None, None, 0.0, 8, None, 0, None, 1 << 40, None, None) == -1
    assert b"16777216 tokens of 128 experts" in lib.frb_last_error()
    assert lib.frb_experts_8bit(None, 0, 3, 100, 2, None, None, None, None, 9000, 40, None, None, 0.0, 8, None, 0, None, 1 << 40, None, None) == -1
    assert b"9000 experts" in lib.frb_last_error()
    # nothing to do is no error
    assert lib.frb_linear_8bit(None, 0, 0, 100, None, None, 33, None, 0, 0, None, 0, None, None) == 0
