"""A cache in 8 bits on the host: what its calls refuse, its pages and tables."""
import importlib

import numpy as np
import pytest
import torch

import fieldrun_b200 as fr
from fieldrun_b200.cache import CacheNeed, SequenceCache
from fieldrun_b200.config.registry import architecture_for
from fieldrun_b200.csrc import ops
from fieldrun_b200.engine.context import StepContext

PAGE = 64
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def store(dtype=INT8, pages=3, heads=2, dim=64, v_heads=None, v_dim=None):
    shape_k, shape_v = (pages, heads, PAGE, dim), (pages, v_heads or heads, PAGE, v_dim or dim)
    return [torch.zeros(shape_k).to(dtype), torch.zeros(shape_k[:3]), torch.zeros(shape_v).to(dtype), torch.zeros(shape_v[:3])]


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def refuses(call, args, options, at, value, match):
    """The call with one of its arguments (a place or a name) put in another's place."""
    args, options = list(args), dict(options)
    if isinstance(at, int):
        args[at] = value
    else:
        options[at] = value
    with pytest.raises(ops.KernelError, match=match):
        call(*args, **options)


HOST = "a CPU tensor was given"


def test_what_writing_refuses():
    k, ks, v, vs = store()
    args = (torch.zeros(3, 6 * 64), None, None, 1e-6, torch.zeros(9, 16), torch.zeros(9, 16), ints(3), ints(3), ints(2, 4),
            torch.zeros(3, 128, dtype=torch.bfloat16), k, ks, v, vs)
    options = dict(num_heads=2, num_kv_heads=2, head_dim=64, rotary_dim=32, interleaved=False)
    with pytest.raises(ops.KernelError, match=HOST):
        ops.qkv_prepare_8bit(*args, **options)
    for at, value, match in [
            (0, torch.zeros(3, 6 * 64 - 4), "projected rows of shape"), (1, torch.ones(128), "come together"),
            (4, None, "rotary tables are missing"), (5, torch.zeros(9, 8), "a rotary table of shape"), (4, torch.zeros(9, 16).double(), "torch.float64"),
            (6, ints(3).long(), "must be torch.int32"), (7, ints(2), "2 slots and a page table"), (8, ints(8), "3 slots and a page table"),
            (9, torch.zeros(3, 128), "query entries of torch.float32"), (9, torch.zeros(3, 64, dtype=torch.bfloat16), "query entries"),
            (10, torch.zeros(3, 2, PAGE, 64), "float8_e4m3fn or int8"), (10, k.to(E4M3), "keys and values alike"), (10, k[:2], "with scales of"),
            (11, ks.double(), "the keys' scales must be"), (11, ks[:, :1], "with scales of"), (12, v[:, :, :32], "pages are"),
            ("head_dim", 48, "8-bit pages of 2 key heads of 64"), ("num_heads", 3, "projected rows of shape"), ("num_kv_heads", 1, "for 1 key heads"),
            ("bias", torch.zeros(6), "a bias of 6"), ("bias", torch.zeros(6 * 64).double(), "must be torch.float32"), ("v_dim", 128, "value heads of 128")]:
        refuses(ops.qkv_prepare_8bit, args, options, at, value, match)
    refuses(ops.qkv_prepare_8bit, (args[0], torch.ones(64), torch.ones(128), *args[3:]), options, "per_head", False, "norm weights of 64 and 128")
    refuses(ops.qkv_prepare_8bit, (*args[:12], *store(pages=4)[2:]), options, "per_head", False, "3 pages of keys and 4 of values")


def test_what_reading_refuses():
    k, ks, v, vs = store(v_heads=1, v_dim=128)
    args = (k, ks, v, vs, ints(2, 4), ints(5), ints(5), ints(2), ints(2), ints(2), torch.zeros(5, 2, PAGE, 64, dtype=torch.bfloat16),
            torch.zeros(5, 1, 128, PAGE, dtype=torch.bfloat16))
    with pytest.raises(ops.KernelError, match=HOST):
        ops.cache_read_8bit(*args)
    for at, value, match in [
            (0, k.float(), "float8_e4m3fn or int8"), (4, ints(8), "slots with"), (5, ints(4), "numbers of pages"), (6, ints(5).long(), "must be torch.int32"),
            (8, ints(3), "2 slots with 3 positions"), (9, ints(1), "1 numbers of new tokens"), (10, torch.zeros(5, 2, PAGE, 64), "keys read back must be"),
            (10, torch.zeros(5, 2, 64, PAGE // 2, dtype=torch.bfloat16), "keys of shape"),
            (11, torch.zeros(5, 1, PAGE, 128, dtype=torch.bfloat16), "values of")]:
        refuses(ops.cache_read_8bit, args, {}, at, value, match)
    odd = store(dim=48)
    with pytest.raises(ops.KernelError, match="known:"):
        ops.cache_read_8bit(*odd, *args[4:10], torch.zeros(5, 2, PAGE, 48, dtype=torch.bfloat16), torch.zeros(5, 2, 48, PAGE, dtype=torch.bfloat16))


def test_what_attention_refuses():
    k, ks, v, vs = store(E4M3)
    args = (torch.zeros(3, 6 * 64, dtype=torch.bfloat16), k, ks, v, vs, ints(5, 4), ints(3), ints(3), torch.zeros(3 * 6 * 64), torch.zeros(3 * 6 * 2),
            torch.zeros(3, 6 * 64, dtype=torch.bfloat16))
    options = dict(num_heads=6, num_kv_heads=2, head_dim=64, scale=0.1, window=None, max_chunks=1)
    with pytest.raises(ops.KernelError, match=HOST):
        ops.attention_decode_8bit(*args, **options)
    for at, value, match in [
            (0, torch.zeros(3, 6 * 64), "queries and outputs are bfloat16"), (0, torch.zeros(3, 5 * 64, dtype=torch.bfloat16), "queries of shape"), (1, k.float(), "float8"),
            (2, ks[:1], "with scales of"), (3, v.to(INT8), "keys and values alike"), (5, ints(5, 4).long(), "the page table, positions and slots must be"), (5, ints(20), "slots and a page table"),
            (6, ints(2), "2 positions"), (7, ints(4), "4 slots"), (8, torch.zeros(3 * 6 * 64).double(), "partial results float32"),
            (10, torch.zeros(3, 6 * 64), "outputs are bfloat16"),
            (10, torch.zeros(3, 64, dtype=torch.bfloat16), "an output of"), ("num_heads", 5, "5 heads over 2"), ("num_kv_heads", 3, "8-bit pages of"),
            ("head_dim", 80, "key heads of 80"), ("v_dim", 128, "8-bit pages of"), ("maps", 3, "with 3 maps"), ("max_chunks", 0, "0 chunks"), ("pieces", 0, "0 pieces"),
            ("window", -1, "a window of -1"), ("keep_first", -1, "-1 first tokens"), ("slopes", torch.zeros(2), "2 numbers for 6 heads"),
            ("sinks", torch.zeros(6).double(), "must be torch.float32"), ("difference", dict(lam=torch.zeros(1), eps=0.1, factor=1.0), "the difference of 1 maps")]:
        refuses(ops.attention_decode_8bit, args, options, at, value, match)


def test_entry_points_refuse_sizes_by_a_message():
    # the C entry points' own checks, which come before anything is launched
    lib = ops.library("cache8")
    assert lib.frb_attention_decode_8bit(*[None] * 5, 0, 1, None, 1, 1, *[None] * 5, 1, 6, 4, 2, 64, 64, 0.1, 0, 0, 0, 1, 1, None, None, 0.0, None, 0.0, 0.0,
                                         1, None, None) == -1
    assert b"6 heads over 4 key heads" in lib.frb_last_error()
    assert lib.frb_attention_decode_8bit(*[None] * 5, 0, 1, None, 1, 1, *[None] * 5, 70_000, 4, 4, 4, 64, 64, 0.1, 0, 0, 0, 1, 1, None, None, 0.0, None, 0.0, 0.0,
                                         1, None, None) == -1
    assert b"exceed the grid" in lib.frb_last_error()
    assert lib.frb_attention_decode_8bit(*[None] * 5, 0, 1 << 24, None, 1, 1, *[None] * 5, 1, 4, 4, 4, 64, 64, 0.1, 0, 0, 0, 1, 1, None, None, 0.0, None, 0.0, 0.0,
                                         1, None, None) == -1
    assert b"exceed a tensor map's rows" in lib.frb_last_error()
    assert lib.frb_cache_read_8bit(*[None] * 4, 5, 1, None, 1, 1, None, None, 1, None, None, None, 1, None, None, 1, 1, 64, 64, None) == -1
    assert b"codes of type 5" in lib.frb_last_error()
    assert lib.frb_qkv_prepare_8bit(None, 0, None, None, 0, 1e-6, None, None, 0, None, None, None, 1, 1, *[None] * 5, 0, 1, 1, 2, 2, 2, 64, 64, 31, 0, 0, 0,
                                    None, 0.0, 1, 0, None, None) == -1
    assert b"rotary_dim 31" in lib.frb_last_error()
    assert lib.frb_qkv_prepare_8bit(4, 0, None, None, 0, 1e-6, None, None, 0, None, None, None, 1, 1, *[None] * 5, 0, 1, 1, 2, 2, 2, 64, 64, 0, 0, 0, 0,
                                    None, 0.0, 1, 0, None, None) == -1
    assert b"rows start on 16 bytes" in lib.frb_last_error()
    assert lib.frb_qkv_prepare_8bit(None, 0, None, None, 0, 1e-6, None, None, 0, None, None, None, 1, 1, *[None] * 5, 0, 1, 1, 900, 2, 2, 64, 64, 0, 0, 0, 0,
                                    None, 0.0, 1, 0, None, None) == -1
    assert b"more than 200 KB" in lib.frb_last_error()


def test_arguments_in_one_struct():
    # the packed entry points read what the ordinary ones get: the same refusals, and numbers beyond 32 bits are an error
    lib = ops.library("cache8")
    attend = [0] * 5 + [0, 1, 0, 1, 1] + [0] * 5 + [1, 6, 4, 2, 64, 64, 0.1, 0, 0, 0, 1, 1, 0, 0, 0.0, 0, 0.0, 0.0, 1, 0]
    read = [0] * 4 + [5, 1, 0, 1, 1, 0, 0, 1, 0, 0, 0, 1, 0, 0, 1, 1, 64, 64]
    write = [0, 0, 0, 0, 0, 1e-6, 0, 0, 0, 0, 0, 0, 1, 1, 0, 0, 0, 0, 0, 0, 1, 1, 2, 2, 2, 64, 64, 31, 0, 0, 0, 0, 0.0, 1, 0, 0]
    for name, args, message in (("frb_attention_decode_8bit", attend, b"6 heads over 4 key heads"), ("frb_cache_read_8bit", read, b"codes of type 5"),
                                ("frb_qkv_prepare_8bit", write, b"rotary_dim 31")):
        assert getattr(lib, name + "_packed")(ops._PACKED[name].pack(*args), None) == -1
        assert message in lib.frb_last_error()
    attend[22] = 1 << 31
    with pytest.raises(ops.KernelError, match="frb_attention_decode_8bit"):
        ops._call("frb_attention_decode_8bit", *attend)


# ------------------------------------------------------------------------------------------------ pages and tables

@pytest.mark.parametrize("codes,dtype", [("int8", INT8), ("float8_e4m3fn", E4M3)])
def test_lines_in_8_bits_have_a_group_of_their_own(codes, dtype):
    needs = [CacheNeed(2, 64), CacheNeed(2, 64, codes=codes), CacheNeed(4, 32, value_dim=64, value_heads=2, window=70, codes=codes), CacheNeed(2, 64, codes=codes)]
    cache = SequenceCache(needs, max_tokens=640, num_slots=3, device="cpu")
    assert [g.lines for g in cache.groups] == [[0], [1, 3], [2]]
    plain, line, other = cache.line(0), cache.line(3), cache.line(2)
    assert plain.key_scales is None and plain.keys.dtype == torch.bfloat16 and tuple(plain.values.shape) == (10, 2, 64, 64)
    assert line.keys.dtype == dtype and tuple(line.values.shape) == (10, 2, 64, 64) and tuple(line.key_scales.shape) == (10, 2, 64)
    assert tuple(other.keys.shape) == (10, 4, 64, 32) and tuple(other.values.shape) == (10, 2, 64, 64) and tuple(other.value_scales.shape) == (10, 2, 64)
    assert other.window == 70 and all(t.is_contiguous() for t in (line.keys, line.values, line.key_scales, other.values))
    s = cache.alloc()
    cache.begin_step([s], [100])
    assert cache.groups[0].table_dev[s, 1] >= 0 and torch.equal(cache.groups[1].table_dev, torch.from_numpy(cache.groups[1].table))
    cache.end_step([s], [100])
    for _ in range(100):
        cache.begin_step([s], [1])
        cache.end_step([s], [1])
    assert cache.groups[2].pool.num_held == 2
    cache.check()
    cache.free(s)
    cache.check()


def test_lines_in_8_bits_are_refused_where_they_make_no_sense():
    with pytest.raises(ValueError, match="'int4'"):
        SequenceCache([CacheNeed(2, 64, codes="int4")], max_tokens=64, device="cpu")
    with pytest.raises(ValueError, match="hold values beside their keys"):
        SequenceCache([CacheNeed(1, 48, value_dim=40, values_in_keys=True, codes="int8")], max_tokens=64, device="cpu")
    writer, reader = CacheNeed(2, 64, window=50, codes="int8"), CacheNeed(2, 64, codes="int8")
    assert writer.shared_with(reader) == reader
    with pytest.raises(ValueError, match="cannot read"):
        writer.shared_with(CacheNeed(2, 64))


@pytest.mark.parametrize("window,chunk,keep_first", [(None, None, 0), (64, None, 0), (1, None, 0), (100, None, 130), (None, 100, 0), (70, 170, 0), (5000, None, 3)])
def test_pages_in_sight(window, chunk, keep_first):
    starts, new = [0, 700, 63, 64, 1000, 129], [1, 5, 1, 200, 0, 64]
    ctx = StepContext.__new__(StepContext)
    ctx.seq_starts, ctx.seq_q_lens, ctx.num_seqs, ctx.device = starts, new, len(starts), torch.device("cpu")
    seqs, numbers, table = ctx.pages_in_sight(window, chunk, keep_first)
    assert seqs.numel() == ctx.visible_pages(window, chunk, keep_first) and table.is_contiguous() and table.dtype == torch.int32
    want = set()
    for b, (start, n) in enumerate(zip(starts, new)):
        for pos in range(start, start + n):
            for key in range(pos + 1):
                lo = max(0, pos - window + 1) if window else 0
                lo = max(lo, pos // chunk * chunk) if chunk else lo
                if key >= lo or (window and key < keep_first):
                    want.add((b, key // PAGE))
    got = list(zip(seqs.tolist(), numbers.tolist()))
    assert set(got) == want and len(got) == len(want)
    for b in range(len(starts)):
        for page in range(table.shape[1]):
            assert int(table[b, page]) == (got.index((b, page)) if (b, page) in want else -1)
    assert ctx.pages_in_sight(window, chunk, keep_first)[2] is table


def build(design, name, dtype, cache_dtype):
    config = importlib.import_module(f"{design}_configs").ALL[name][0]
    arch = architecture_for(config, "config")
    return fr.build_model(arch, arch.config_from_dict(config, "config"), dtype, cache_dtype)


@pytest.mark.parametrize("design,name", [("tiny", "b"), ("tiny", "d"), ("bamasun", "C"), ("fotanex", "C"), ("bakasun", "C"), ("duzinex", "C"), ("kifunex", "C")])
def test_models_with_a_cache_in_8_bits(design, name):
    for given, codes in (("int8", "int8"), (torch.float8_e4m3fn, "float8_e4m3fn"), (None, ""), ("", "")):
        model = build(design, name, "bfloat16", given)
        needs = model.cache_needs()
        assert any(n.kv_heads for n in needs) and all(n.codes == (codes if n.kv_heads else "") for n in needs)
        assert ("cache8" in model.kernel_groups()) == bool(codes)
        assert model.replayable


def test_models_that_cannot_hold_their_cache_in_8_bits_say_so():
    with pytest.raises(ValueError, match="for bfloat16 models"):
        build("tiny", "d", "float32", "int8")
    with pytest.raises(ValueError, match=r"\(16, 16\)"):
        build("tiny", "a", "bfloat16", "int8")
    with pytest.raises(ValueError, match="latent_attention.*model's dtype only"):
        build("depelix", "C", "bfloat16", "float8_e4m3fn")
    for name in ("int4", "bfloat16", torch.uint8, 8):
        with pytest.raises(ValueError, match="a cache of type"):
            build("tiny", "d", "bfloat16", name)
