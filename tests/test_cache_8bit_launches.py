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


# ------------------------------------------------------------------------------------------------ pages read back in portions

def step_of(starts, new):
    from fieldrun_b200.engine.context import StepContext
    ctx = StepContext.__new__(StepContext)
    ctx.seq_starts, ctx.seq_q_lens, ctx.num_seqs, ctx.device, ctx._tiles = starts, new, len(starts), torch.device("cpu"), {}
    ctx.max_q_len, ctx.max_kv_len, ctx.is_decode = max(new), max(a + b for a, b in zip(starts, new)), False
    return ctx


@pytest.mark.parametrize("options", [(None, None, 0), (100, None, 130), (None, 100, 0)])
@pytest.mark.parametrize("most", [1, 4, 12, 13, 1000])
def test_pages_in_sight_in_portions(options, most):
    starts, new = [0, 700, 63, 64, 1000, 129, 5000, 0], [1, 5, 1, 200, 0, 64, 70, 0]
    ctx = step_of(starts, new)
    seqs, numbers, whole = ctx.pages_in_sight(*options)
    portions, table = ctx.sight_portions(*options, most)
    # the same pages in the same order, whole sequences, every sequence in one portion
    assert torch.equal(torch.cat([p.page_seq for p in portions]), seqs) and torch.equal(torch.cat([p.page_index for p in portions]), numbers)
    assert portions[0].first_seq == 0 and portions[-1].end_seq == len(new) and all(a.end_seq == b.first_seq for a, b in zip(portions, portions[1:]))
    at = 0
    for p in portions:
        assert p.page_seq.numel() <= most or p.page_seq.unique().numel() == 1
        assert all(p.first_seq <= b < p.end_seq for b in p.page_seq.tolist()) and sum(new[p.first_seq:p.end_seq]) > 0
        inside = whole[p.first_seq:p.end_seq]
        assert torch.equal(table[p.first_seq:p.end_seq], torch.where(inside >= 0, inside - at, inside))
        at += p.page_seq.numel()
        for rows in (16, 128):
            got, all_tiles = ctx.query_tiles(rows, p), ctx.query_tiles(rows)
            keep = (all_tiles[0] >= p.first_seq) & (all_tiles[0] < p.end_seq)
            assert all(torch.equal(a, b[keep]) for a, b in zip(got, all_tiles))
        assert ctx.tokens_of(p) == slice(sum(new[:p.first_seq]), sum(new[:p.end_seq]))
    # no two portions that would have gone together
    assert all(a.page_seq.numel() + int((b.page_seq == b.page_seq[0]).sum()) > most for a, b in zip(portions, portions[1:]))


@pytest.mark.parametrize("new", [[2, 1, 70, 1, 1], [1, 3, 1, 1, 1]])
def test_a_mixed_step_reads_back_no_more_than_its_room_at_a_time(new, monkeypatch):
    """One prompt among sequences of one token each must not turn all of their histories into bfloat16 pages at once."""
    part, held, made = mixer("tiny", "d"), {}, []
    monkeypatch.setattr("fieldrun_b200.parts.attention.READ_BACK_BYTES", 20 * PAGE * 2 * 2 * (2 * 64))        # 20 pages of 2 heads of 64
    starts = [640, 1000, 500, 64, 4000]
    ctx = step_of(starts, new)
    tokens = sum(new)
    ints = torch.zeros(tokens, dtype=torch.int32)
    ctx.tok_pos = ctx.tok_slot = ctx.tok_seq = ctx.seq_slot = ctx.seq_start = ctx.seq_q_len = ctx.cu_q_len = ints

    def buffer(name, shape, dtype):
        held[name] = max(held.get(name, 0), shape[0])
        return torch.empty(shape, dtype=dtype)
    ctx.buffer = buffer
    monkeypatch.setattr(ops, "cache_read_8bit", lambda *args: made.append((args[5], args[6], args[10].shape[0], args[11].shape[0])))
    names = ("attention_prefill_tc", "attention_prefill_mma")
    for name in names:
        monkeypatch.setattr(ops, name, lambda q, k, v, table, tile_seq, tile_q0, *args, **options: made.append((k.shape[0], tile_seq.tolist())))
    rows = torch.zeros(tokens, part.q_width, dtype=torch.bfloat16)
    part.attend(ctx, rows, LineView(None, None, None, None, None), rows.clone())
    # 11 | 16 | 9 (or 8) + 2 | 63: as many as there is room for, and one sequence that needs more by itself
    third = -(-(500 + new[2]) // PAGE) + 2
    assert [read[2] for read in made[::2]] == [11, 16, third, 63] and held["attention.keys"] == held["attention.values"] == 63
    assert [sorted(set(tiles)) for _, tiles in made[1::2]] == [[0], [1], [2, 3], [4]] and [n for n, _ in made[1::2]] == [11, 16, third, 63]


def test_the_general_kernel_gets_a_portions_own_tokens(monkeypatch):
    # a cap together with slopes, which no other kernel takes
    part, made = mixer("tiny", "d"), []
    part.softcap, part.slopes = 5.0, torch.ones(part.q_heads)
    monkeypatch.setattr("fieldrun_b200.parts.attention.READ_BACK_BYTES", 1)
    ctx = step_of([640, 64, 500], [2, 1, 70])
    ctx.tok_pos = ctx.tok_slot = ctx.seq_slot = ctx.seq_start = ctx.seq_q_len = ctx.cu_q_len = torch.arange(73, dtype=torch.int32)
    ctx.tok_seq = torch.tensor([0] * 2 + [1] + [2] * 70, dtype=torch.int32)
    ctx.buffer = lambda name, shape, dtype: torch.empty(shape, dtype=dtype)
    monkeypatch.setattr(ops, "cache_read_8bit", lambda *args: None)
    monkeypatch.setattr(ops, "attention_generic", lambda q, k, v, table, tok_pos, tok_slot, out, *, gate, **options: made.append((q, tok_pos.tolist(), set(tok_slot.tolist()), out, gate)))
    rows = torch.zeros(73, part.q_width, dtype=torch.bfloat16)
    out, gate = torch.zeros(73, part.out_width, dtype=torch.bfloat16), torch.zeros(73, part.num_heads)
    part.attend(ctx, rows, LineView(None, None, None, None, None), out, gate)
    bounds = [(0, 2), (2, 3), (3, 73)]
    assert [(positions, seqs) for _, positions, seqs, _, _ in made] == [(list(range(a, b)), {i}) for i, (a, b) in enumerate(bounds)]
    for (q, _, _, o, g), (a, b) in zip(made, bounds):
        assert all(t.data_ptr() == whole[a:].data_ptr() and t.shape[0] == b - a and t.is_contiguous() for t, whole in ((q, rows), (o, out), (g, gate)))
