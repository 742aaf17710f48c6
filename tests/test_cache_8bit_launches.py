"""What is asked of the kernels over a cache in 8 bits, on the host: calls are looked at and not made."""
import importlib
import types

import pytest
import torch

import fieldrun_b200 as fr
from fieldrun_b200.cache import LineView
from fieldrun_b200.config.registry import architecture_for
from fieldrun_b200.csrc import ops
from fieldrun_b200.parts.attention import GQAAttention

PAGE = 64


@pytest.fixture
def calls(monkeypatch):
    """The calls of entry points, with tensors on the host for those of the device."""
    made = []
    monkeypatch.setattr(ops, "_call", lambda name, *args: made.append((name, args)))
    monkeypatch.setattr(ops, "_ptr", lambda t: 0)
    monkeypatch.setattr(ops, "_addresses", lambda *tensors: [0] * len(tensors))
    monkeypatch.setattr(ops, "tc_status", lambda device: None)
    return made


def attend(**options):
    def ints(*shape):
        return torch.zeros(shape, dtype=torch.int32)
    codes, scales = torch.zeros(3, 2, PAGE, 64, dtype=torch.int8), torch.zeros(3, 2, PAGE)
    rows = torch.zeros(3, 6 * 64, dtype=torch.bfloat16)
    ops.attention_decode_8bit(rows, codes, scales, codes, scales, ints(5, 4), ints(3), ints(3), torch.zeros(3 * 6 * 64), torch.zeros(3 * 6 * 2), rows.clone(),
                              num_heads=6, num_kv_heads=2, head_dim=64, scale=0.1, window=None, max_chunks=1, **options)


def test_pages_are_read_ahead_of_the_kernel_before_only_where_the_caller_says_so(calls):
    """The kernel before may be the one that writes a prompt's rows into those pages."""
    for options in ({}, {"pages_final": False}, {"pages_final": True}):
        attend(**options)
    assert [(name, args[-2]) for name, args in calls] == [("frb_attention_decode_8bit", 0), ("frb_attention_decode_8bit", 0), ("frb_attention_decode_8bit", 1)]


def mixer(design, name, codes="int8"):
    """An attention part of a model with a cache in 8 bits."""
    config = importlib.import_module(f"{design}_configs").ALL[name][0]
    arch = architecture_for(config, "config")
    model = fr.build_model(arch, arch.config_from_dict(config, "config"), "bfloat16", codes)
    return next(block.mixer for block in model.blocks if isinstance(block.mixer, GQAAttention))


def test_a_step_of_single_tokens_says_that_older_pages_are_final(monkeypatch):
    part, made = mixer("tiny", "d"), []
    monkeypatch.setattr(ops, "attention_decode_8bit", lambda *args, **options: made.append(options))
    ctx = types.SimpleNamespace(is_decode=True, max_kv_len=700, num_seqs=2, seq_start=None, seq_slot=None, tok_slot=None,
                                buffer=lambda name, shape, dtype: torch.empty(shape, dtype=dtype))
    rows = torch.zeros(2, part.q_width, dtype=torch.bfloat16)
    part.attend(ctx, rows, LineView(None, None, None, None, None), rows.clone())
    assert len(made) == 1 and made[0]["pages_final"] is True
