"""The kernels of a cache in 8 bits against plain float64: rows written, pages read back, one token's attention."""
import numpy as np
import pytest
import torch

import cache_8bit_plain as plain
from fieldrun_b200.csrc import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 64
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
SIZES = [(32, 32), (32, 64), (64, 64), (64, 128), (96, 96), (128, 128)]


def generator(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ rows written

class Written:
    """One call of qkv_prepare_8bit on random rows, and the same in float64."""

    def __init__(self, positions, dtype, heads=6, kv_heads=2, dim=64, v_dim=None, v_heads=None, norm="none", rotary=0, interleaved=False,
                 bias=False, q_temp=None, values_from_keys=False, in_dtype=torch.float32, weight_dtype=torch.float32, seed=1, rows=None):
        v_dim, v_heads = v_dim or dim, v_heads or kv_heads
        gen = generator(seed)
        tokens = len(positions)
        width = (heads + kv_heads) * dim + (0 if values_from_keys else v_heads * v_dim)
        qkv = rows if rows is not None else (torch.randn(tokens, width, generator=gen, device=DEV)
                                             * torch.exp(torch.randn(width, generator=gen, device=DEV))).to(in_dtype)
        self.qkv, self.tokens, self.dtype = qkv, tokens, dtype
        weights = dict(none=(0, 0), per_head=(dim, dim), full_width=(heads * dim, kv_heads * dim))[norm]
        qw, kw = ((1 + 0.2 * torch.randn(n, generator=gen, device=DEV)).to(weight_dtype) if n else None for n in weights)
        b = torch.randn(width, generator=gen, device=DEV) if bias else None
        cos = sin = None
        if rotary:
            angle = torch.rand(max(positions) + 1, rotary // 2, generator=gen, device=DEV) * 6.28
            cos, sin = torch.cos(angle), torch.sin(angle)
        slots = 1 + max(positions) // PAGE, tokens + 2
        table = torch.full((slots[1], slots[0]), -1, dtype=torch.int32, device=DEV)
        order = torch.randperm(tokens + 3, generator=gen, device=DEV)
        slot = torch.randperm(slots[1], generator=gen, device=DEV)[:tokens]
        for i, pos in enumerate(positions):
            table[slot[i], pos // PAGE] = order[i]
        self.k = torch.full((tokens + 3, kv_heads, PAGE, dim), 1.0, device=DEV).to(dtype)
        self.v = torch.full((tokens + 3, v_heads, PAGE, v_dim), 1.0, device=DEV).to(dtype)
        self.ks = torch.full((tokens + 3, kv_heads, PAGE), 7.0, device=DEV)
        self.vs = torch.full((tokens + 3, v_heads, PAGE), 7.0, device=DEV)
        self.q = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device=DEV)
        self.where = [(int(order[i]), pos % PAGE) for i, pos in enumerate(positions)]
        self.args = (qkv, qw, kw, 1e-6, cos, sin, ints(positions), slot.to(torch.int32), table, self.q, self.k, self.ks, self.v, self.vs)
        self.options = dict(num_heads=heads, num_kv_heads=kv_heads, num_v_heads=v_heads, head_dim=dim, v_dim=v_dim, rotary_dim=rotary,
                            interleaved=interleaved, per_head=norm == "per_head", bias=b, q_temp=q_temp, values_from_keys=values_from_keys)
        # in float64, with the size that the rotation's rounding is relative to beside every entry
        x = qkv.double().cpu().numpy() + (b.double().cpu().numpy() if bias else 0.0)
        q, k = x[:, :heads * dim], x[:, heads * dim:(heads + kv_heads) * dim]
        self.want_v = (k if values_from_keys else x[:, (heads + kv_heads) * dim:]).reshape(tokens, v_heads, v_dim)
        parts = []
        for part, n, w in ((q, heads, qw), (k, kv_heads, kw)):
            if norm == "per_head":
                part = part.reshape(tokens, n, dim)
            if norm != "none":
                part = part / np.sqrt((part * part).mean(-1, keepdims=True) + 1e-6) * w.double().cpu().numpy()
            parts.append(part.reshape(tokens, n, dim).copy())
        q, k = parts
        if q_temp:
            q = q * (1 + q_temp[0] * np.log(np.floor((np.array(positions) + 1) / q_temp[1]) + 1))[:, None, None]
        self.want_q, self.size_q = self.rotated(q, positions, cos, sin, rotary, interleaved)
        self.want_k, self.size_k = self.rotated(k, positions, cos, sin, rotary, interleaved)

    @staticmethod
    def rotated(x, positions, cos, sin, rotary, interleaved):
        size = np.abs(x)
        if not rotary:
            return x, size
        c, s = (t.double().cpu().numpy()[positions][:, None, :] for t in (cos, sin))
        half = rotary // 2
        one, two = (np.arange(half) * 2, np.arange(half) * 2 + 1) if interleaved else (np.arange(half), np.arange(half) + half)
        out, size = x.copy(), size.copy()
        out[..., one], out[..., two] = x[..., one] * c - x[..., two] * s, x[..., two] * c + x[..., one] * s
        size[..., one] = size[..., two] = np.abs(x[..., one]) + np.abs(x[..., two])
        return out, size

    def run(self):
        ops.qkv_prepare_8bit(*self.args, **self.options)
        return self

    # float32 arithmetic: a sum of up to 2^13 squares in runs of a few dozen and a tree (2^-19 of it at most, half of that in its root),
    # a square root, a quotient and four products (2^-24 each), a rotation (2^-23 of both terms): below 2^-19 of the terms' size
    SLACK = 2.0 ** -19

    def check(self):
        heads, dim = self.options["num_heads"], self.options["head_dim"]
        q = self.q.double().cpu().numpy().reshape(self.tokens, heads, dim)
        assert (np.abs(q - self.want_q) <= 2.0 ** -8 * np.abs(self.want_q) + 2 * self.SLACK * self.size_q + 1e-37).all()
        for codes, scales, want, size in ((self.k, self.ks, self.want_k, self.size_k), (self.v, self.vs, self.want_v, np.abs(self.want_v))):
            got, scale = plain.numbers(codes), scales.double().cpu().numpy()
            limit = plain.LIMIT[self.dtype]
            slack = self.SLACK * size.max(-1, keepdims=True)
            top = np.abs(want).max(-1, keepdims=True)
            for i, (page, place) in enumerate(self.where):
                assert (np.abs(scale[page, :, place] - top[i, :, 0] / limit) <= 2 * slack[i, :, 0] / limit).all()
                # the code of what lies within the slack of the exact entry
                y = want[i] / top[i] * limit
                off = 4 * slack[i] / top[i] * limit
                lo, hi = plain.to_grid(y - off, self.dtype), plain.to_grid(y + off, self.dtype)
                assert ((got[page, :, place] >= np.clip(lo, -limit, limit)) & (got[page, :, place] <= np.clip(hi, -limit, limit))).all()
        return self

    def check_untouched(self):
        """Every other place holds what it held."""
        for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
            keep = torch.ones(codes.shape[0], PAGE, dtype=torch.bool, device=DEV)
            for page, place in self.where:
                keep[page, place] = False
            assert (codes.float().transpose(1, 2)[keep] == 1.0).all() and (scales.transpose(1, 2)[keep] == 7.0).all()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim,v_dim", SIZES)
def test_written_head_sizes(dim, v_dim, dtype):
    Written([0, 63, 64, 700, 5], dtype, dim=dim, v_dim=v_dim, rotary=dim, norm="per_head").run().check().check_untouched()


@pytest.mark.parametrize("norm", ["none", "per_head", "full_width"])
@pytest.mark.parametrize("rotary,interleaved", [(0, False), (64, False), (32, True), (20, False), (18, True), (2, False), (44, True)])
def test_written_norms_and_rotations(norm, rotary, interleaved):
    Written([3, 64, 130], E4M3, dim=64, norm=norm, rotary=rotary, interleaved=interleaved, bias=True).run().check().check_untouched()


@pytest.mark.parametrize("heads,kv_heads,v_heads,dim,v_dim", [(48, 8, 8, 128, 128), (1, 1, 1, 32, 32), (7, 7, 7, 96, 96), (32, 8, 4, 64, 128), (12, 3, 3, 64, 64)])
def test_written_head_counts(heads, kv_heads, v_heads, dim, v_dim):
    norm = "full_width" if v_heads == kv_heads else "none"
    Written([9, 10, 200], INT8, heads=heads, kv_heads=kv_heads, v_heads=v_heads, dim=dim, v_dim=v_dim, norm=norm, rotary=dim // 2).run().check().check_untouched()


@pytest.mark.parametrize("tokens", [1, 2, 296, 297, 700])
def test_written_token_counts(tokens):
    Written([(37 * i) % 500 for i in range(tokens)], E4M3, heads=4, kv_heads=2, dim=128, norm="full_width", rotary=64).run().check().check_untouched()


def test_written_types_and_options():
    Written([5, 6], E4M3, dim=128, norm="full_width", in_dtype=torch.bfloat16, weight_dtype=torch.bfloat16, rotary=64).run().check()
    Written([5, 6, 8191], INT8, dim=64, norm="per_head", weight_dtype=torch.bfloat16, q_temp=(0.1, 64), rotary=64).run().check()
    Written([5, 6], INT8, dim=128, rotary=64, values_from_keys=True, bias=True).run().check().check_untouched()
    Written([70, 6], E4M3, dim=96, rotary=96, interleaved=True, values_from_keys=True).run().check().check_untouched()
    w = Written([70, 6], E4M3, dim=64, rotary=32)
    w.options["tables_final"] = True
    w.run().check().check_untouched()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_written_rows_of_unusual_numbers(dtype):
    rows = torch.randn(6, 4 * 64, device=DEV, generator=generator(2))
    rows[0, 128:] = 0.0                                          # keys and values of zeros
    rows[1, 130], rows[1, 200] = float("inf"), float("nan")      # rows that are not finite
    rows[2, 128:] *= 1e-32                                       # below what is kept
    rows[3, 128:] *= 1e35
    rows[4, 128:192] = -3.0                                      # all entries at the limit
    rows[5, 128:] *= 1e-20
    w = Written([0, 1, 2, 3, 4, 5], dtype, heads=2, kv_heads=1, dim=64, rows=rows).run()
    for i, (page, place) in enumerate(w.where):
        for codes, scales, part in ((w.k, w.ks, rows[i, 128:192]), (w.v, w.vs, rows[i, 192:])):
            got, scale = codes[page, 0, place].float(), scales[page, 0, place]
            if i == 1:
                assert torch.isnan(scale) and (got == 0).all()
            elif i in (0, 2):
                assert scale == 0 and (got == 0).all()
            else:
                want, ref = plain.store_rows(part.double().cpu().numpy()[None], dtype)
                assert abs(scale.item() - ref[0]) <= 2.0 ** -22 * ref[0]
                assert (got.abs().max() == plain.LIMIT[dtype]) and np.abs(got.cpu().numpy() - want[0]).max() <= plain.LIMIT[dtype] / 14
    assert (w.k[w.where[4][0], 0, w.where[4][1]].float() == -plain.LIMIT[dtype]).all()


def test_written_tokens_without_a_place_write_nothing():
    w = Written([0, 64, 10, 20, 30], E4M3, dim=64)
    positions, slots, table = w.args[6], w.args[7], w.args[8]
    positions[0], slots[1] = -5, 10_000
    positions[2] = PAGE * table.shape[1]
    table[slots[3].long(), 0] = -1
    table[slots[4].long(), 0] = w.k.shape[0]
    w.run()
    w.where = []
    w.check_untouched()


def test_written_twice_is_the_same_bits_and_a_row_does_not_depend_on_the_others():
    positions = [3, 4, 500, 64, 65]
    a = Written(positions, E4M3, heads=48, kv_heads=8, dim=128, norm="full_width", rotary=64).run()
    b = Written(positions, E4M3, heads=48, kv_heads=8, dim=128, norm="full_width", rotary=64).run()
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.vs, b.vs) and torch.equal(a.q, b.q)
    alone = Written(positions, E4M3, heads=48, kv_heads=8, dim=128, norm="full_width", rotary=64)
    alone.args = (alone.qkv[2:3].contiguous(), *alone.args[1:6], alone.args[6][2:3].contiguous(), alone.args[7][2:3].contiguous(), alone.args[8],
                  alone.q[2:3], *alone.args[10:])
    alone.run()
    page, place = a.where[2]
    assert torch.equal(a.k.view(torch.uint8)[page, :, place], alone.k.view(torch.uint8)[page, :, place])
    assert torch.equal(a.ks[page, :, place], alone.ks[page, :, place]) and torch.equal(a.q[2], alone.q[2])


# ------------------------------------------------------------------------------------------------ pages read back

@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim,v_dim,kv_heads,v_heads", [(32, 32, 1, 1), (32, 64, 4, 4), (64, 64, 3, 3), (64, 128, 4, 2), (96, 96, 2, 2), (128, 128, 8, 8)])
def test_pages_read_back(dim, v_dim, kv_heads, v_heads, dtype):
    gen = generator(dim + v_dim)
    starts, new = [0, 100, 60, 0, 200], [1, 28, 5, 64, 0]
    lengths = [a + b for a, b in zip(starts, new)]
    pages, slots = 40, 9
    k, ks = plain.random_store(gen, pages, kv_heads, dim, dtype)
    v, vs = plain.random_store(gen, pages, v_heads, v_dim, dtype)
    if dtype == E4M3:
        k.view(torch.uint8)[30:] = 0x7f                          # NaN where no sequence looks
        v.view(torch.uint8)[30:] = 0xff
    ks[30:] = float("nan")
    vs[30:] = float("inf")
    slot = torch.randperm(slots, generator=gen, device=DEV)[:5]
    table = torch.full((slots, 5), 35, dtype=torch.int32, device=DEV)
    order = torch.randperm(30, generator=gen, device=DEV)
    at = 0
    asked = []
    for b, n in enumerate(lengths):
        held = -(-n // PAGE)
        table[slot[b], :held] = order[at:at + held].to(torch.int32)
        at += held
        asked += [(b, p) for p in range(held + 1)]               # one page behind the last, too
    asked += [(1, 0), (4, 0)]                                    # a page twice, and one given back
    table[slot[4], 0] = -1
    asked += [(-1, 0), (5, 0), (0, -1), (0, 5)]                  # sequences and pages that do not exist
    keys = torch.full((len(asked), kv_heads, PAGE, dim), float("nan"), dtype=torch.bfloat16, device=DEV)
    values = torch.full((len(asked), v_heads, v_dim, PAGE), float("nan"), dtype=torch.bfloat16, device=DEV)
    ops.cache_read_8bit(k, ks, v, vs, table, ints([a for a, _ in asked]), ints([b for _, b in asked]), slot.to(torch.int32), ints(starts),
                        ints(new), keys, values)
    for n, (b, index) in enumerate(asked):
        page = int(table[slot[b], index]) if 0 <= b < 5 and 0 <= index < 5 else -1
        there = max(0, min(PAGE, lengths[b] - PAGE * index)) if page >= 0 else 0
        want_k = torch.zeros(kv_heads, PAGE, dim, device=DEV)
        want_v = torch.zeros(v_heads, PAGE, v_dim, device=DEV)
        want_k[:, :there] = k[page].float()[:, :there] * ks[page][:, :there, None]
        want_v[:, :there] = v[page].float()[:, :there] * vs[page][:, :there, None]
        assert torch.equal(keys[n], want_k.to(torch.bfloat16)), (n, b, index)
        assert torch.equal(values[n], want_v.to(torch.bfloat16).transpose(1, 2)), (n, b, index)


def test_no_pages_to_read():
    k, ks = plain.random_store(generator(1), 2, 1, 64, INT8)
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    ops.cache_read_8bit(k, ks, k, ks, ints([[0]]), empty, empty, ints([0]), ints([0]), ints([1]),
                        torch.empty(0, 1, PAGE, 64, dtype=torch.bfloat16, device=DEV), torch.empty(0, 1, 64, PAGE, dtype=torch.bfloat16, device=DEV))


# ------------------------------------------------------------------------------------------------ one token's attention

class Attended:
    """One call of attention_decode_8bit over random pages, and the same in float64."""

    def __init__(self, positions, dtype, heads=6, kv_heads=2, dim=64, v_dim=None, maps=1, seed=3, q_size=1.0, k_spread=0.5, pages_more=3, **options):
        v_dim = v_dim or dim
        gen = generator(seed)
        self.heads, self.kv_heads, self.maps, self.dim, self.v_dim, self.dtype = heads, kv_heads, maps, dim, v_dim, dtype
        self.v_heads = kv_heads // maps
        counts = [p // PAGE + 1 for p in positions]
        pages = sum(counts) + pages_more
        self.k, self.ks = plain.random_store(gen, pages, kv_heads, dim, dtype, k_spread)
        self.v, self.vs = plain.random_store(gen, pages, self.v_heads, v_dim, dtype, 0.3)
        self.slots = torch.randperm(len(positions) + 2, generator=gen, device=DEV)[:len(positions)].to(torch.int32)
        self.table = torch.full((len(positions) + 2, max(counts) + 1), -1, dtype=torch.int32, device=DEV)
        order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        at = 0
        for i, n in enumerate(counts):
            self.table[self.slots[i].long(), :n] = order[at:at + n]
            at += n
        self.unused = order[at:].long()
        self.positions = positions
        self.q = (q_size * torch.randn(len(positions), heads * dim, generator=gen, device=DEV)).to(torch.bfloat16)
        self.options = dict(num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, v_dim=v_dim, scale=dim ** -0.5, window=None, maps=maps,
                            max_chunks=-(-(max(max(positions), 0) + 1) // 256))
        self.options.update(options)
        if maps == 2:
            self.options["difference"] = dict(lam=torch.full((1,), 0.35, device=DEV), eps=1e-5, factor=0.7)
        rows = len(positions) * heads * self.options["max_chunks"]
        self.part_o = torch.full((rows * v_dim,), float("nan"), device=DEV)
        self.part_ml = torch.full((rows * 2,), float("nan"), device=DEV)
        self.out = torch.full((len(positions), heads // maps * v_dim), float("nan"), dtype=torch.bfloat16, device=DEV)

    def run(self):
        ops.attention_decode_8bit(self.q, self.k, self.ks, self.v, self.vs, self.table, ints(self.positions), self.slots, self.part_o,
                                  self.part_ml, self.out, **self.options)
        ops.tc_status_check(self.q.device)
        return self

    def rows_of(self, i, codes, scales):
        n = self.positions[i] // PAGE + 1
        pages = self.table[self.slots[i].long(), :n].long()
        x = plain.numbers(codes.view(torch.uint8)[pages].view(codes.dtype)) * scales[pages].double().cpu().numpy()[..., None]
        return x.transpose(1, 0, 2, 3).reshape(x.shape[1], n * PAGE, -1)

    def check(self):
        o = self.options
        arrays = {n: o[n].double().cpu().numpy() if o.get(n) is not None else None for n in ("slopes", "sinks")}
        got = self.out.double().cpu().numpy().reshape(len(self.positions), self.heads // self.maps, self.v_dim)
        for i, position in enumerate(self.positions):
            if position < 0:
                assert (got[i] == 0).all()
                continue
            q = self.q[i].double().cpu().numpy().reshape(self.heads, self.dim)
            want, size, top, reach, span = plain.attend(q, self.rows_of(i, self.k, self.ks), self.rows_of(i, self.v, self.vs), position,
                                                  scale=o["scale"], group=self.heads // self.kv_heads, maps=self.maps, window=o["window"],
                                                  chunk=o.get("chunk"), keep_first=o.get("keep_first", 0), softcap=o.get("softcap"), **arrays)
            d = o.get("difference")
            more = dict(lam=float(d["lam"].double()), eps=d["eps"], factor=d["factor"]) if d else {}
            want, bound = plain.output_bound(want, size, top, reach, span, position, dim=self.dim, codes=self.dtype, group=self.heads // self.kv_heads, maps=self.maps,
                                             softcap=o.get("softcap"), slopes=arrays["slopes"], **more)
            off = np.abs(got[i] - want)
            assert np.isfinite(got[i]).all() and (off <= bound).all(), (i, position, float((off / bound).max()))
        return self


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim,v_dim", SIZES)
def test_attention_head_sizes(dim, v_dim, dtype):
    Attended([0, 1, 62, 63, 64, 65, 255, 256, 777], dtype, dim=dim, v_dim=v_dim).run().check()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (7, 1), (8, 1), (9, 1), (16, 1), (17, 1), (48, 2), (33, 1), (48, 8)])
def test_attention_group_sizes(heads, kv_heads, dtype):
    Attended([5, 300, 130], dtype, heads=heads, kv_heads=kv_heads, dim=128).run().check()
    Attended([70, 3], dtype, heads=heads, kv_heads=kv_heads, dim=32).run().check()


MASKS = [dict(window=1), dict(window=64), dict(window=65), dict(window=300), dict(window=10_000), dict(chunk=1), dict(chunk=64), dict(chunk=100),
         dict(chunk=1000), dict(window=100, chunk=170), dict(window=90, keep_first=1), dict(window=64, keep_first=64),
         dict(window=300, keep_first=130), dict(window=100, keep_first=5000)]


@pytest.mark.parametrize("options", MASKS, ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()))
@pytest.mark.parametrize("pieces", [None, 1, 3, 29, 1000])
def test_attention_masks(options, pieces):
    Attended([0, 63, 64, 200, 999, 1300, 511], INT8, heads=12, kv_heads=4, dim=64, pieces=pieces, **options).run().check()
    Attended([1300, 40, 1023], E4M3, heads=10, kv_heads=1, dim=128, pieces=pieces, **options).run().check()


def test_attention_scores_with_everything():
    gen = generator(9)
    for heads, kv_heads, dim in ((12, 2, 64), (24, 2, 128), (20, 1, 96)):
        extra = dict(slopes=2.0 ** torch.linspace(-1, -9, heads, device=DEV), sinks=2 * torch.randn(heads, generator=gen, device=DEV), softcap=5.0)
        for names in (["slopes"], ["sinks"], ["softcap"], ["slopes", "sinks"], ["slopes", "sinks", "softcap"]):
            Attended([0, 64, 700], E4M3, heads=heads, kv_heads=kv_heads, dim=dim, window=400, keep_first=3, **{n: extra[n] for n in names}).run().check()
            Attended([90, 300], INT8, heads=heads, kv_heads=kv_heads, dim=dim, chunk=128, **{n: extra[n] for n in names}).run().check()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim,v_dim,heads,kv_heads", [(64, 128, 32, 8), (32, 64, 8, 2), (128, 128, 4, 4), (64, 64, 40, 2)])
def test_attention_of_two_maps(dim, v_dim, heads, kv_heads, dtype):
    Attended([0, 100, 640], dtype, heads=heads, kv_heads=kv_heads, dim=dim, v_dim=v_dim, maps=2).run().check()
    Attended([700, 30], dtype, heads=heads, kv_heads=kv_heads, dim=dim, v_dim=v_dim, maps=2, window=200, keep_first=70, softcap=10.0).run().check()


def test_attention_long_sequences_and_the_split():
    for pieces in (None, 1, 5, 8, 64, 1776):
        Attended([16000, 3, 9000], E4M3, heads=12, kv_heads=2, dim=128, pieces=pieces).run().check()


@pytest.mark.parametrize("chunks", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("pieces", [None, 1, 7, 200])
def test_attention_many_short_sequences(chunks, pieces):
    # partial results have little room or none: the line is cut between key heads only, or into few pieces a head
    positions = [-1 if i % 11 == 5 else (257 * i * i + 63 * (i % 3)) % (256 * chunks) for i in range(90)]
    a = Attended(positions, E4M3, heads=24, kv_heads=12, dim=64, pieces=pieces, max_chunks=chunks).run().check()
    index = [0, 1, 1, 1, 40, 41, 41, 89, 89]                       # with rows repeated
    a.positions = [positions[i] for i in index]
    a.q, a.slots, a.out = a.q[index].contiguous(), a.slots[index].contiguous(), a.out[index].contiguous()
    a.run().check()
    assert torch.equal(a.out[1], a.out[2]) and torch.equal(a.out[2], a.out[3]) and torch.equal(a.out[5], a.out[6]) and torch.equal(a.out[7], a.out[8])
    Attended(positions[:40], INT8, heads=18, kv_heads=1, dim=128, pieces=pieces, max_chunks=chunks, window=150, keep_first=70).run().check()


@pytest.mark.parametrize("chunks,pieces", [(1, None), (1, 50), (4, None), (4, 3000)])
def test_attention_thousands_of_sequences(chunks, pieces):
    # more rows than 64 groups of 32
    positions = [-1 if i % 7 == 3 else (i * 37) % 130 + (600 if chunks == 4 and i % 97 == 0 else 0) for i in range(2500)]
    Attended(positions, E4M3, heads=2, kv_heads=1, dim=32, pieces=pieces, max_chunks=chunks).run().check()


@pytest.mark.parametrize("chunks,pieces", [(1, 9), (4, 1), (4, 333), (12, 40), (12, None)])
def test_attention_of_a_row_repeated_many_times(chunks, pieces):
    # over the bounds of 32 rows, at the end and in the middle
    lengths = [256 * chunks - 5, 100, -1, 70]
    counts = [3, 69, 1, 60]
    a = Attended(lengths, INT8, heads=12, kv_heads=6, dim=64, pieces=pieces, max_chunks=chunks)
    index = torch.tensor([i for i, n in enumerate(counts) for _ in range(n)], device=DEV)
    a.positions = [lengths[int(i)] for i in index]
    a.q, a.slots, a.out = a.q[index].contiguous(), a.slots[index].contiguous(), a.out[index].contiguous()
    a.part_o, a.part_ml = (x.reshape(len(lengths), -1)[index].reshape(-1).contiguous() for x in (a.part_o, a.part_ml))
    a.run().check()
    for i in range(len(lengths)):
        rows = a.out[index == i]
        assert torch.equal(rows, rows[:1].expand_as(rows))


def test_attention_sharp_scores():
    # one key has nearly all the weight, at any place, and scores of hundreds: the running maximum moves by much
    for seed in range(4):
        Attended([1500, 700], INT8, heads=8, kv_heads=1, dim=128, q_size=30.0, seed=seed).run().check()
        Attended([1500, 700], E4M3, heads=16, kv_heads=1, dim=64, q_size=30.0, k_spread=1.0, seed=seed).run().check()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_attention_values_of_unequal_sizes(dtype):
    # values whose sizes differ by 2^60 within a page and from page to page, a huge one with hardly any weight among them, and rows of zeros
    for heads in (6, 12):
        a = Attended([900, 200, 70], dtype, heads=heads, kv_heads=1, dim=64)
        gen = generator(17)
        a.vs *= 2.0 ** torch.randint(-12, 12, a.vs.shape, generator=gen, device=DEV)
        a.run().check()
        a.vs[:, :, ::3] = 0.0
        a.ks[:, :, 5] = 0.0
        a.run().check()
        a.vs *= 2.0 ** torch.randint(-60, 40, (a.vs.shape[0], 1, 1), generator=gen, device=DEV)
        a.run().check()
        a.vs[:] = 0.0
        a.run()
        assert (a.out == 0).all()


def test_attention_queries_of_unequal_sizes():
    a = Attended([300, 70], E4M3, heads=12, kv_heads=2, dim=128)
    q = a.q.view(2, 12, 128)
    q[:, 0] = 0.0
    q[:, 1] *= 2.0 ** -120
    q[:, 2] *= 2.0 ** 5
    q[0, 3, 1:] *= 2.0 ** -14
    a.run().check()
    a = Attended([300, 70], INT8, heads=12, kv_heads=2, dim=128)
    a.q *= 2.0 ** -60
    a.ks *= 2.0 ** 60
    a.run().check()


def test_attention_ignores_what_lies_behind_and_before_the_keys_it_sees():
    for options in (dict(), dict(window=70, keep_first=5), dict(chunk=100)):
        for dtype in (E4M3, INT8):
            a = Attended([100, 333, 63, 0], dtype, heads=10, kv_heads=2, dim=64, **options).run().check()
            clean = a.out.clone()
            for i, pos in enumerate(a.positions):
                lo = max(0, pos - 69) if "window" in options else pos // 100 * 100 if "chunk" in options else 0
                hidden = [k for k in range((pos // PAGE + 1) * PAGE) if k > pos or (k < lo and k >= options.get("keep_first", 0))]
                for key in hidden:
                    page = int(a.table[a.slots[i].long(), key // PAGE])
                    if dtype == E4M3:
                        a.k.view(torch.uint8)[page, :, key % PAGE] = 0x7f
                        a.v.view(torch.uint8)[page, :, key % PAGE] = 0xff
                    a.ks[page, :, key % PAGE] = float("nan")
                    a.vs[page, :, key % PAGE] = float("inf") if key % 2 else float("nan")
            a.k.view(torch.uint8)[a.unused] = 0x7f
            a.ks[a.unused] = float("nan")
            a.run()
            assert torch.equal(a.out, clean)


def test_attention_a_row_that_is_not_finite_shows_where_it_is_seen():
    a = Attended([300, 310], E4M3, heads=6, kv_heads=2, dim=64, window=100)
    page = int(a.table[a.slots[0].long(), 250 // PAGE])
    a.ks[page, 1, 250 % PAGE] = float("nan")
    a.run()
    got = a.out.view(2, 6, 64)
    assert torch.isnan(got[0, 3:]).all() and torch.isfinite(got[0, :3]).all() and torch.isfinite(got[1]).all()
    for options in (dict(), dict(softcap=9.0)):
        a = Attended([300], INT8, heads=6, kv_heads=2, dim=64, **options)
        page = int(a.table[a.slots[0].long(), 0])
        a.ks[page, 0] = float("nan")
        a.run()
        assert torch.isnan(a.out.view(6, 64)[:3]).all() and torch.isfinite(a.out.view(6, 64)[3:]).all()
        a.ks[page, 0] = 1.0
        a.vs[page, 1, 7] = float("nan")
        a.run()
        assert torch.isnan(a.out.view(6, 64)[3:]).all() and torch.isfinite(a.out.view(6, 64)[:3]).all()


def test_attention_of_sequences_and_pages_that_are_not_there():
    a = Attended([-1, 200, 100, -7], E4M3, heads=6, kv_heads=2, dim=64, sinks=torch.zeros(6, device=DEV)).run().check()
    # a slot that does not exist gives zeros, too
    a.slots[1] = 100
    a.run()
    assert (a.out[1] == 0).all()
    # pages that the table does not have hold no keys: the rest is attended over
    a = Attended([700], INT8, heads=6, kv_heads=2, dim=64)
    row = a.slots[0].long()
    full = a.table[row].clone()
    a.table[row, 2] = -1
    a.table[row, 5] = a.k.shape[0] + 5
    a.run()
    q = a.q[0].double().cpu().numpy().reshape(6, 64)
    got = a.out.clone()
    a.table[row] = full
    keep = np.ones(11 * PAGE, dtype=bool)
    keep[2 * PAGE:3 * PAGE] = keep[5 * PAGE:6 * PAGE] = False
    keep[701:] = False
    k, v = a.rows_of(0, a.k, a.ks)[:, keep], a.rows_of(0, a.v, a.vs)[:, keep]
    want, size, *_ = plain.attend(q, k, v, int(keep.sum()) - 1, scale=0.125, group=3)
    assert (np.abs(got.double().cpu().numpy().reshape(6, 64) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * size).all()
    a.table[row] = -1
    a.run()
    assert (a.out == 0).all()


def test_attention_refuses_too_little_room_and_tensors_in_pieces():
    a = Attended([100, 700], E4M3, heads=6, kv_heads=2, dim=64, pieces=1)
    for name, value in (("part_o", a.part_o[:-1]), ("part_ml", a.part_ml[:-1])):
        kept = getattr(a, name)
        setattr(a, name, value)
        with pytest.raises(ops.KernelError, match="room for"):
            a.run()
        setattr(a, name, kept)
    kept, a.out = a.out, a.out.t().contiguous().t()
    with pytest.raises(ops.KernelError, match="not contiguous"):
        a.run()
    a.out = kept
    a.q = a.q.cpu()
    with pytest.raises(ops.KernelError, match="a CPU tensor"):
        a.run()


@pytest.mark.parametrize("name", ["part_o", "part_ml", "out", "q", "ks", "vs", "k", "v"])
def test_attention_refuses_tensors_off_their_boundaries(name):
    a = Attended([100, 700], E4M3, heads=6, kv_heads=2, dim=64)
    held = getattr(a, name)
    wide = torch.empty(held.numel() + 1, dtype=held.dtype, device=DEV)
    setattr(a, name, wide[1:].view(held.shape))
    with pytest.raises(ops.KernelError, match="start on"):
        a.run()


def test_attention_more_keys_than_the_launch_is_sized_for_are_reported():
    a = Attended([100, 1000], E4M3, heads=6, kv_heads=2, dim=64)
    a.options["max_chunks"] = 2
    with pytest.raises(ops.KernelError, match="more keys than the launch was sized for"):
        a.run()
    a.options["max_chunks"] = 4
    a.run().check()


def test_attention_twice_is_the_same_bits():
    for lengths in ([2000, 300, 64], [9000] * 20):
        a = Attended(lengths, INT8, heads=12, kv_heads=2, dim=128).run()
        first = a.out.clone()
        a.run()
        assert torch.equal(a.out, first)


@pytest.mark.parametrize("pieces", [None, 1, 7, 40, 5000])
@pytest.mark.parametrize("times", [2, 3, 9])
def test_attention_of_repeated_rows_is_the_same_bits(times, pieces):
    # a recorded step repeats its last row; here rows in the middle are repeated, too, among them one without tokens
    for lengths, heads, kv_heads, options in (([700, 64, 5000, -1, 333], 12, 2, {}), ([6000, 4000], 6, 6, dict(window=3000, keep_first=70)), ([20000], 20, 1, {})):
        counts = [1 + (i % 2) * (times - 1) for i in range(len(lengths) - 1)] + [times]
        a = Attended(lengths, E4M3, heads=heads, kv_heads=kv_heads, dim=64, pieces=pieces, **options)
        index = torch.tensor([i for i, n in enumerate(counts) for _ in range(n)], device=DEV)
        a.positions = [lengths[int(i)] for i in index]
        a.q, a.slots, a.out = a.q[index].contiguous(), a.slots[index].contiguous(), a.out[index].contiguous()
        a.part_o, a.part_ml = (x.reshape(len(lengths), -1)[index].reshape(-1).contiguous() for x in (a.part_o, a.part_ml))
        a.run()
        for i in range(len(lengths)):
            rows = a.out[index == i]
            assert torch.equal(rows, rows[:1].expand_as(rows))
        a.check()


def test_attention_beyond_32_bits():
    # a store of more than 2^32 bytes of keys, the sequence's pages at its ends
    pages, heads = 66_000, 8
    k = torch.zeros(pages, heads, PAGE, 128, dtype=torch.int8, device=DEV)
    v = torch.zeros(pages, heads, PAGE, 128, dtype=torch.int8, device=DEV)
    ks, vs = torch.zeros(pages, heads, PAGE, device=DEV), torch.zeros(pages, heads, PAGE, device=DEV)
    a = Attended([500], INT8, heads=8, kv_heads=8, dim=128)
    place = torch.tensor([0, 65_999, 32_768, 65_998, 33_000, 65_000, 1, 60_000], device=DEV)
    held = a.table[a.slots[0].long(), :8].long()
    for big, small in ((k, a.k), (v, a.v), (ks, a.ks), (vs, a.vs)):
        big[place] = small[held]
    a.k, a.v, a.ks, a.vs = k, v, ks, vs
    a.table[a.slots[0].long(), :8] = place.to(torch.int32)
    a.run().check()
    keys = torch.empty(8, heads, PAGE, 128, dtype=torch.bfloat16, device=DEV)
    values = torch.empty(8, heads, 128, PAGE, dtype=torch.bfloat16, device=DEV)
    ops.cache_read_8bit(k, ks, v, vs, a.table, ints([0] * 8), ints(list(range(8))), a.slots, ints([500]), ints([1]), keys, values)
    assert torch.equal(keys[1], (k[65_999].float() * ks[65_999][..., None]).to(torch.bfloat16))
    # a row written there
    w = Written([70], INT8, heads=8, kv_heads=8, dim=128)
    w.args[8][w.args[7].long(), 1] = 65_999
    w.args = (*w.args[:10], k, ks, v, vs)
    w.run()
    w.k, w.ks, w.v, w.vs = (x[65_998:] for x in (k, ks, v, vs))
    w.where = [(1, 6)]
    w.check()


# ------------------------------------------------------------------------------------------------ streams and graphs

def test_recorded_and_on_another_stream():
    def both():
        return Written([70, 6], E4M3, heads=6, kv_heads=2, dim=64, rotary=64), Attended([600, 70], E4M3, heads=6, kv_heads=2, dim=64)
    w, a = both()
    w.run(), a.run()
    want = [t.clone().view(torch.uint8) for t in (w.k, w.vs, w.q, a.out)]
    w2, a2 = both()
    pos = ints(a2.positions)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w2.run()
        ops.attention_decode_8bit(a2.q, a2.k, a2.ks, a2.v, a2.vs, a2.table, pos, a2.slots, a2.part_o, a2.part_ml, a2.out, **a2.options)
    side.synchronize()
    assert all(torch.equal(x, t.view(torch.uint8)) for x, t in zip(want, (w2.k, w2.vs, w2.q, a2.out)))
    w3, a3 = both()
    keys = torch.empty(3, 2, PAGE, 64, dtype=torch.bfloat16, device=DEV)
    values = torch.empty(3, 2, 64, PAGE, dtype=torch.bfloat16, device=DEV)
    seq, index, starts, new = ints([0, 0, 1]), ints([0, 9, 1]), ints([600, 70]), ints([1, 1])
    ops.cache_read_8bit(a.k, a.ks, a.v, a.vs, a.table, seq, index, a.slots, starts, new, keys, values)
    read = keys.clone(), values.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w3.run_ = ops.qkv_prepare_8bit(*w3.args, **w3.options)
        ops.attention_decode_8bit(a3.q, a3.k, a3.ks, a3.v, a3.vs, a3.table, pos, a3.slots, a3.part_o, a3.part_ml, a3.out, **a3.options)
        ops.cache_read_8bit(a3.k, a3.ks, a3.v, a3.vs, a3.table, seq, index, a3.slots, starts, new, keys, values)
    for _ in range(3):
        for t in (w3.q, a3.out, keys, values, a3.part_o, a3.part_ml):
            t.fill_(float("nan"))
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, t.view(torch.uint8)) for x, t in zip(want, (w3.k, w3.vs, w3.q, a3.out)))
    assert torch.equal(keys, read[0]) and torch.equal(values, read[1])


def test_rows_written_and_attended_one_after_the_other():
    # a prompt's rows and a token's attention over them, nothing in between: the attention waits for all of its pages
    tokens, heads, kv_heads, dim = 300, 12, 4, 64
    gen = generator(31)
    table = torch.randperm(5, generator=gen, device=DEV).to(torch.int32).view(1, 5)
    positions, zeros = torch.arange(tokens, dtype=torch.int32, device=DEV), torch.zeros(tokens, dtype=torch.int32, device=DEV)
    qkv = [torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=gen, device=DEV) for _ in range(20)]
    results = []
    for wait in (True, False):
        for rows in qkv:
            k, v = (torch.full((5, kv_heads, PAGE, dim), 3, dtype=torch.int8, device=DEV) for _ in range(2))
            ks, vs = (torch.full((5, kv_heads, PAGE), 9.0, device=DEV) for _ in range(2))
            q = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device=DEV)
            part_o, part_ml = torch.empty(heads, 2, dim, device=DEV), torch.empty(heads, 2, 2, device=DEV)
            last, out = torch.randn(1, heads * dim, generator=generator(5), device=DEV).to(torch.bfloat16), torch.empty(1, heads * dim, dtype=torch.bfloat16, device=DEV)
            position = ints([tokens - 1])
            torch.cuda.synchronize()
            ops.qkv_prepare_8bit(rows, None, None, 1e-6, None, None, positions, zeros, table, q, k, ks, v, vs, num_heads=heads, num_kv_heads=kv_heads,
                                 head_dim=dim, rotary_dim=0, interleaved=False)
            if wait:
                torch.cuda.synchronize()
            ops.attention_decode_8bit(last, k, ks, v, vs, table, position, zeros[:1], part_o, part_ml, out, num_heads=heads, num_kv_heads=kv_heads,
                                      head_dim=dim, scale=dim ** -0.5, window=None, max_chunks=2, pages_final=wait)
            ops.tc_status_check(out.device)
            results.append(out)
    for a, b in zip(results, results[len(qkv):]):
        assert torch.equal(a, b)


def test_attention_refuses_a_lambda_without_an_entry():
    a = Attended([100, 70], E4M3, heads=8, kv_heads=4, dim=64, maps=2)
    a.options["difference"]["lam"] = torch.empty(0, device=DEV)
    with pytest.raises(ops.KernelError, match="lambda"):
        a.run()


@pytest.mark.parametrize("tokens,pieces", [(300, None), (300, 7), (2000, None)])
def test_a_prompt_written_and_attended_without_a_word(tokens, pieces):
    # as above with no option given: attention reads what the kernel right before it wrote
    heads, kv_heads, dim = 12, 4, 64
    gen = generator(33)
    pages = -(-tokens // PAGE)
    table = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32).view(1, pages)
    positions, zeros, position = torch.arange(tokens, dtype=torch.int32, device=DEV), torch.zeros(tokens, dtype=torch.int32, device=DEV), ints([tokens - 1])
    last = torch.randn(1, heads * dim, generator=gen, device=DEV).to(torch.bfloat16)
    chunks = -(-tokens // 256)
    part_o, part_ml = torch.empty(heads, chunks, dim, device=DEV), torch.empty(heads, chunks, 2, device=DEV)
    for _ in range(10):
        rows = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=gen, device=DEV)
        results = []
        for wait in (True, False):
            k, v = (torch.full((pages, kv_heads, PAGE, dim), 3, dtype=torch.int8, device=DEV) for _ in range(2))
            ks, vs = (torch.full((pages, kv_heads, PAGE), 9.0, device=DEV) for _ in range(2))
            q, out = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device=DEV), torch.empty(1, heads * dim, dtype=torch.bfloat16, device=DEV)
            torch.cuda.synchronize()
            ops.qkv_prepare_8bit(rows, None, None, 1e-6, None, None, positions, zeros, table, q, k, ks, v, vs, num_heads=heads, num_kv_heads=kv_heads,
                                 head_dim=dim, rotary_dim=0, interleaved=False)
            if wait:
                torch.cuda.synchronize()
            ops.attention_decode_8bit(last, k, ks, v, vs, table, position, zeros[:1], part_o, part_ml, out, num_heads=heads, num_kv_heads=kv_heads,
                                      head_dim=dim, scale=dim ** -0.5, window=None, max_chunks=chunks, pieces=pieces)
            ops.tc_status_check(out.device)
            results.append(out)
        assert torch.equal(*results)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("ratio", [2.0 ** 7, 2.0 ** 10, 2.0 ** 12, 2.0 ** 20])
@pytest.mark.parametrize("dim,heads,kv_heads,pieces", [(128, 12, 2, None), (128, 10, 1, 5), (64, 12, 4, 9), (96, 12, 2, None), (32, 4, 4, None)])
def test_attention_scores_beside_a_large_query_entry(dim, heads, kv_heads, pieces, ratio, dtype):
    # one entry of every query head is `ratio` times the largest of the others, and the keys are zero there: what it
    # multiplies is nothing, and the other entries count to their last bit
    a = Attended([900, 70], dtype, heads=heads, kv_heads=kv_heads, dim=dim, pieces=pieces, q_size=4.0, k_spread=0.0, seed=41)
    q = a.q.view(2, heads, dim)
    for head in range(heads):
        place = (7 * (head // (heads // kv_heads)) + 3) % dim                # the heads of a key head share the place
        q[:, head, place] = 0.0
        q[:, head, place] = ratio * q[:, head].abs().amax(-1)
        a.k.view(torch.uint8)[:, head // (heads // kv_heads), :, place] = 0
    a.run()
    got = a.out.double().cpu().numpy().reshape(2, heads, a.v_dim)
    for i, position in enumerate(a.positions):
        want, size, top, reach, _ = plain.attend(a.q[i].double().cpu().numpy().reshape(heads, dim), a.rows_of(i, a.k, a.ks), a.rows_of(i, a.v, a.vs),
                                                 position, scale=dim ** -0.5, group=heads // kv_heads)
        # queries as they are: no term for their rounding (and none for their largest entry)
        want, bound = plain.output_bound(want, size, top, reach, 0.0, position, dim=dim, group=heads // kv_heads, codes=None)
        off = np.abs(got[i] - want)
        assert (off <= bound).all(), (i, float((off / bound).max()))
