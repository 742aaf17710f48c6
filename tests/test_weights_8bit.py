"""Models with weights in 8 bits on the host: which parts take them, what is refused."""
import importlib

import pytest
import torch

import fieldrun_b200 as fr
from fieldrun_b200.config.registry import architecture_for
from fieldrun_b200.csrc import ops
from fieldrun_b200.parts.linear import Weight8, linear

DESIGNS = [("tiny", "a"), ("tiny", "d"), ("bamasun", "C"), ("fotanex", "C"), ("depelix", "C"), ("bakasun", "C"), ("duzinex", "C"), ("kifunex", "B")]


def build(design, name, dtype="bfloat16", **more):
    config = importlib.import_module(f"{design}_configs").ALL[name][0]
    arch = architecture_for(config, "config")
    return fr.build_model(arch, arch.config_from_dict(config, "config"), dtype, **more)


@pytest.mark.parametrize("design,name", DESIGNS)
def test_models_with_weights_in_8_bits(design, name):
    plain = build(design, name)
    for given, codes in (("int8", "int8"), (torch.int8, "int8"), (None, ""), ("", "")):
        model = build(design, name, weight_dtype=given)
        took = [part for part in model.all_parts() if part.weight_codes]
        assert bool(took) == bool(codes) and all(part.weight_codes == codes for part in took)
        assert ("products8" in model.kernel_groups()) == bool(codes)
        assert set(plain.kernel_groups()) <= set(model.kernel_groups())
        assert model.replayable == plain.replayable
        assert [need.name for need in model.tensor_needs()] == [need.name for need in plain.tensor_needs()]


def test_with_a_cache_in_8_bits_beside():
    model = build("tiny", "d", cache_dtype="int8", weight_dtype="int8")
    assert {"cache8", "products8"} <= set(model.kernel_groups()) and any(n.codes for n in model.cache_needs())


def test_models_that_cannot_hold_their_weights_in_8_bits_say_so():
    with pytest.raises(ValueError, match="for bfloat16 models"):
        build("tiny", "d", "float32", weight_dtype="int8")
    for name in ("int4", "bfloat16", torch.uint8, 8):
        with pytest.raises(ValueError, match="weights of type"):
            build("tiny", "d", weight_dtype=name)

    with pytest.raises(ValueError, match="weights in .int4."):
        build("tiny", "d").blocks[0].mixer.store_weights_as("int4")


def test_a_weight_of_many_experts():
    weight = Weight8(40, 100, "cpu", parts=2, experts=3)
    assert weight.codes.shape == (3, 2, 48, 128) and weight.scales.shape == (3, 2, 48) and (weight.features, weight.inner) == (40, 100)
    assert weight.pair[0] is weight.codes and not weight.codes.any()
    with pytest.raises(ops.KernelError, match="a CPU tensor was given"):
        weight.put(0, torch.zeros(40, 100), torch.zeros(40, 100))
    with pytest.raises(ops.KernelError, match="not \\[1, 1, 48, 128\\]"):
        weight.put(0, torch.zeros(40, 100))
    with pytest.raises(ops.KernelError, match="a CPU tensor was given"):
        linear(torch.zeros(2, 100), Weight8(40, 100, "cpu"))
