"""A cache in 8 bits on the host: what its calls refuse, its pages and tables."""
import pytest
import torch

from fieldrun_b200.csrc import ops

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
            (4, None, "rotary tables are missing"), (5, torch.zeros(9, 8), "a rotary table of shape"), (4, torch.zeros(9, 16).double(), "must be torch.float32"),
            (6, ints(3).long(), "positions must be torch.int32"), (7, ints(2), "2 slots for 3 tokens"), (8, ints(8), "positions and"),
            (9, torch.zeros(3, 128), "queries must be torch.bfloat16"), (9, torch.zeros(3, 64, dtype=torch.bfloat16), "query entries"),
            (10, torch.zeros(3, 2, PAGE, 64), "float8_e4m3fn or int8"), (10, k.to(E4M3), "keys and values alike"), (10, k[:2], "with scales of"),
            (11, ks.double(), "the keys' scales must be"), (11, ks[:, :1], "with scales of"), (12, v[:, :, :32], "pages are"),
            ("head_dim", 48, "known:"), ("num_heads", 3, "projected rows of shape"), ("num_kv_heads", 1, "projected rows of shape"),
            ("bias", torch.zeros(6), "a bias of 6"), ("bias", torch.zeros(6 * 64).double(), "must be torch.float32"), ("v_dim", 128, "projected rows")]:
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
            (0, torch.zeros(3, 6 * 64), "queries must be"), (0, torch.zeros(3, 5 * 64, dtype=torch.bfloat16), "queries of shape"), (1, k.float(), "float8"),
            (2, ks[:1], "with scales of"), (3, v.to(INT8), "keys and values alike"), (5, ints(5, 4).long(), "the page table must be"), (5, ints(20), "positions and"),
            (6, ints(2), "2 positions"), (7, ints(4), "4 slots"), (8, torch.zeros(3 * 6 * 64 - 1), "room for"), (9, torch.zeros(35), "room for"),
            (8, torch.zeros(3 * 6 * 64).double(), "must be torch.float32"), (10, torch.zeros(3, 6 * 64), "the attention output must be"),
            (10, torch.zeros(3, 64, dtype=torch.bfloat16), "an output of"), ("num_heads", 5, "5 heads over 2"), ("num_kv_heads", 3, "8-bit pages of"),
            ("head_dim", 80, "known:"), ("v_dim", 128, "8-bit pages of"), ("maps", 3, "with 3 maps"), ("max_chunks", 0, "0 chunks"), ("chunks_per_block", 0, "0 per block"),
            ("window", -1, "a window of -1"), ("keep_first", -1, "-1 first tokens"), ("slopes", torch.zeros(2), "2 numbers for 6 heads"),
            ("sinks", torch.zeros(6).double(), "must be torch.float32"), ("difference", dict(lam=torch.zeros(1), eps=0.1, factor=1.0), "the difference of 1 maps")]:
        refuses(ops.attention_decode_8bit, args, {**options, "chunks_per_block": 1} if at != "chunks_per_block" else options, at, value, match)


def test_entry_points_refuse_sizes_by_a_message():
    # the C entry points' own checks, which come before anything is launched
    lib = ops.library("cache8")
    assert lib.frb_attention_decode_8bit(*[None] * 5, 0, 1, None, 1, 1, *[None] * 5, 1, 6, 4, 2, 64, 64, 0.1, 0, 0, 0, 1, 1, None, None, 0.0, None, 0.0, 0.0,
                                         None, None) == -1
    assert b"6 heads over 4 key heads" in lib.frb_last_error()
    assert lib.frb_attention_decode_8bit(*[None] * 5, 0, 1, None, 1, 1, *[None] * 5, 70_000, 4, 4, 4, 64, 64, 0.1, 0, 0, 0, 1, 1, None, None, 0.0, None, 0.0, 0.0,
                                         None, None) == -1
    assert b"exceed the grid" in lib.frb_last_error()
    assert lib.frb_attention_decode_8bit(*[None] * 5, 0, 1 << 24, None, 1, 1, *[None] * 5, 1, 4, 4, 4, 64, 64, 0.1, 0, 0, 0, 1, 1, None, None, 0.0, None, 0.0, 0.0,
                                         None, None) == -1
    assert b"exceed a tensor map's rows" in lib.frb_last_error()
    assert lib.frb_cache_read_8bit(*[None] * 4, 5, 1, None, 1, 1, None, None, 1, None, None, None, 1, None, None, 1, 1, 64, 64, None) == -1
    assert b"codes of type 5" in lib.frb_last_error()
    assert lib.frb_qkv_prepare_8bit(None, 0, None, None, 0, 1e-6, None, None, 0, None, None, None, 1, 1, *[None] * 5, 0, 1, 1, 2, 2, 2, 64, 64, 31, 0, 0, 0,
                                    None, 0.0, 1, 0, None) == -1
    assert b"rotary_dim 31" in lib.frb_last_error()
    assert lib.frb_qkv_prepare_8bit(4, 0, None, None, 0, 1e-6, None, None, 0, None, None, None, 1, 1, *[None] * 5, 0, 1, 1, 2, 2, 2, 64, 64, 0, 0, 0, 0,
                                    None, 0.0, 1, 0, None) == -1
    assert b"whole group of four" in lib.frb_last_error()
    assert lib.frb_qkv_prepare_8bit(None, 0, None, None, 0, 1e-6, None, None, 0, None, None, None, 1, 1, *[None] * 5, 0, 1, 1, 900, 2, 2, 64, 64, 0, 0, 0, 0,
                                    None, 0.0, 1, 0, None) == -1
    assert b"more than 200 KB" in lib.frb_last_error()
