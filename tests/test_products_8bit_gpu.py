"""Products in 8-bit integers on the device against plain ones in 64 bits: rows as codes, a linear layer, a gated block, routed experts."""
import pytest
import torch

import plain_products_8bit as plain
from fieldrun_b200.csrc import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    torch.cuda.synchronize()
    ops.tc_status_check(torch.device("cuda:0"))
    ops.tc_status_check("cuda")


def generator(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows_of(gen, rows, inner, dtype=BF16):
    x = torch.randn((rows, inner), generator=gen, device=DEV)
    return (x * torch.exp(torch.randn((rows, 1), generator=gen, device=DEV))).to(dtype)


def linear(x, w, s, features, dtype=F32, out=None, **more):
    out = torch.full((x.shape[0], features), float("nan"), dtype=dtype, device=DEV) if out is None else out
    ops.linear_8bit(x, w, s, out, **more)
    return out


# ------------------------------------------------------------------------------------------------ rows

def stored(x):
    codes = torch.full((x.shape[0], plain.up(x.shape[1], 128)), 99, dtype=torch.int8, device=DEV)
    scales = torch.full((x.shape[0],), 99.0, device=DEV)
    ops.rows_8bit(x, codes, scales)
    return codes, scales


def check_rows(x):
    codes, scales = stored(x)
    want, step = plain.codes_of(x)
    assert torch.equal(codes[:, :x.shape[1]].double(), want)
    assert not codes[:, x.shape[1]:].any()
    assert ((scales.double() - step[:, 0]).abs() <= plain.U * step[:, 0]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, inner", [(1, 1), (1, 7), (3, 8), (2, 127), (5, 128), (300, 129), (700, 1000), (1, 4096), (9, 4104), (301, 4097), (2, 16385), (2, 20000),
                                         (1, 131072)])
def test_rows(rows, inner, dtype):
    check_rows(rows_of(generator(rows + inner), rows, inner, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_with_values_in_the_middle_of_two_codes(dtype):
    # whole numbers of half a step: with a largest entry of 127 * 2^n every odd number of halves is a middle; others have middles at a half of it
    gen = generator(3)
    halves = torch.randint(-254, 255, (64, 512), generator=gen, device=DEV).float() / 2
    halves[:, 0] = 127
    x = halves * torch.exp2(torch.arange(-32.0, 32.0, device=DEV))[:, None]
    check_rows(x.to(dtype) if dtype == F32 else x.to(dtype))
    top = torch.rand((200, 1), generator=gen, device=DEV).to(dtype).float() + 1
    check_rows((top * torch.tensor([[1.0, 0.5, -0.5, -1.0, 0.25, 0.0]], device=DEV)).to(dtype))


def test_rows_at_the_ends_of_the_types():
    tiny, huge = 2.0 ** -96, 3.0e38
    x = torch.tensor([[0.0, 0.0, -0.0], [tiny, -tiny / 2, 0.0], [tiny * 0.99, 0.0, 0.0], [1e-40, 1e-45, 0.0], [huge, -huge, huge / 2], [1e-30, 1.0, -1e-30]], device=DEV)
    check_rows(x)
    codes, scales = stored(x)
    assert scales[[0, 2, 3]].tolist() == [0.0, 0.0, 0.0] and not codes[[0, 2, 3]].any()
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = torch.ones((3, 300), device=DEV)
        y[1, 255] = bad
        codes, scales = stored(y)
        assert scales.isnan().tolist() == [False, True, False] and not codes[1].any() and (codes[[0, 2], :300] == 127).all()


def test_a_weight_is_its_rows():
    gen = generator(5)
    gate, up = (torch.randn((33, 100), generator=gen, device=DEV).to(BF16) for _ in range(2))
    codes, scales = ops.weight_8bit(gate, up)
    for part, c, s in zip((gate, up), codes[0], scales[0]):
        want, step = plain.codes_of(part)
        assert torch.equal(c[:33, :100].double(), want) and not c[33:].any() and not c[:, 100:].any() and not s[33:].any()
        assert torch.allclose(s[:33].double(), step[:, 0], rtol=2.0 ** -24, atol=0.0)
    many, many_scales = torch.zeros((3, *codes.shape[1:]), dtype=torch.int8, device=DEV), torch.zeros((3, *scales.shape[1:]), device=DEV)
    ops.weight_8bit(gate, up, codes=many[1:2], scales=many_scales[1:2])
    assert torch.equal(many[1], codes[0]) and torch.equal(many_scales[1], scales[0]) and not many[0].any() and not many[2].any()


# ------------------------------------------------------------------------------------------------ a linear layer

@pytest.mark.parametrize("rows", [1, 2, 8, 9, 31, 64, 127, 128, 129, 200, 256, 257, 1000])
@pytest.mark.parametrize("inner, features", [(1, 1), (100, 15), (128, 16), (129, 257), (1024, 100), (640, 1000), (4096, 48)])
def test_linear(rows, inner, features):
    gen = generator(rows * 7 + inner)
    dtype, result = ((BF16, F32), (F32, BF16), (BF16, BF16), (F32, F32))[(rows + inner) % 4]
    x = rows_of(gen, rows, inner, dtype)
    codes, scales, w, s = plain.random_weight(gen, 1, 1, features, inner, DEV)
    exact, bound = plain.product(x, codes[0, 0], scales[0, 0])
    plain.agree(linear(x, w, s, features, result), exact, bound, (rows, inner, features))


@pytest.mark.parametrize("rows, inner, features", [(1, 6144, 8192), (40, 4096, 4096), (128, 2048, 6144), (300, 1000, 20000), (2000, 1536, 2048), (3000, 200, 1999)])
def test_linear_at_sizes_of_models(rows, inner, features):
    gen = generator(rows)
    x = rows_of(gen, rows, inner)
    codes, scales, w, s = plain.random_weight(gen, 1, 1, features, inner, DEV)
    exact, bound = plain.product(x, codes[0, 0], scales[0, 0])
    plain.agree(linear(x, w, s, features), exact, bound)


@pytest.mark.parametrize("rows", [1, 130])
def test_the_longest_sum_of_the_largest_codes(rows):
    inner = ops.EIGHT_BIT_MOST_INNER
    x = torch.ones((rows, inner), device=DEV)
    x[:, ::2] = -1
    codes = torch.full((1, 1, 32, inner), 127.0, device=DEV, dtype=torch.float64)
    codes[0, 0, 0::3, ::2] = -127
    codes[0, 0, 1::3, 1::2] = -127
    w, s = plain.laid_out(codes, torch.ones((1, 1, 32), device=DEV))
    exact, bound = plain.product(x, codes[0, 0], s[0, 0, :32])
    assert exact.abs().max() * 127 >= 127 ** 2 * inner * 0.999
    plain.agree(linear(x, w, s, 32), exact, bound)


@pytest.mark.parametrize("features, inner", [(100, 300), (2048, 1024)])
def test_a_rows_results_are_its_own(features, inner):
    gen = generator(1)
    x = rows_of(gen, 700, inner)
    _, _, w, s = plain.random_weight(gen, 1, 1, features, inner, DEV)
    whole = linear(x, w, s, features)
    for first, count in [(0, 1), (3, 5), (128, 64), (200, 128), (5, 300), (699, 1)]:
        assert torch.equal(linear(x[first:first + count], w, s, features), whole[first:first + count])


def test_rows_of_nan_stay_by_themselves():
    gen = generator(2)
    for rows in (5, 300):
        x = rows_of(gen, rows, 200)
        _, _, w, s = plain.random_weight(gen, 1, 1, 40, 200, DEV)
        good = linear(x, w, s, 40)
        x[2, 199], x[4, 0] = float("nan"), float("inf")
        got = linear(x, w, s, 40)
        bad = torch.zeros(rows, dtype=torch.bool, device=DEV)
        bad[[2, 4]] = True
        assert got[bad].isnan().all() and torch.equal(got[~bad], good[~bad])
    x = torch.zeros((5, 200), device=DEV)
    assert not linear(x, w, s, 40).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("features", [64, 40, 36, 33])
def test_results_at_any_place_and_nothing_beside_them(rows, dtype, features):
    gen = generator(rows)
    codes, scales, w, s = plain.random_weight(gen, 1, 1, features, 256, DEV)
    flat = rows_of(gen, rows + 1, 256).reshape(-1)
    for place in (0, 1, 4, 8):
        x = flat[place:place + rows * 256].view(rows, 256)            # from an odd place on, too
        room = torch.full((rows * features + 64,), 7.0, dtype=dtype, device=DEV)
        out = room[place:place + rows * features].view(rows, features)
        ops.linear_8bit(x, w, s, out)
        exact, bound = plain.product(x, codes[0, 0], scales[0, 0])
        plain.agree(out, exact, bound)
        assert (room[:place] == 7).all() and (room[place + rows * features:] == 7).all()


def test_results_beyond_32_bits_of_places():
    gen = generator(4)
    rows, features = 70_001, 32_000
    x = rows_of(gen, rows, 128)
    codes, scales, w, s = plain.random_weight(gen, 1, 1, features, 128, DEV)
    out = linear(x, w, s, features, BF16)
    for some in (slice(0, 200), slice(67_000, 67_200), slice(rows - 200, rows)):
        exact, bound = plain.product(x[some], codes[0, 0], scales[0, 0])
        plain.agree(out[some], exact, bound)


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_scales_at_the_ends_of_the_range(rows):
    # a token's scale of 2^96 and more, a channel's of 2^-100: no product on the way is infinite or loses places
    gen = generator(rows)
    codes, _, w, s = plain.random_weight(gen, 1, 1, 64, 512, DEV)
    x = torch.randn((rows, 512), generator=gen, device=DEV)
    for of_x, of_w in ((2.0 ** 120, 2.0 ** -100), (2.0 ** -90, 2.0 ** 110), (2.0 ** -60, 2.0 ** -50), (2.0 ** 30, 2.0 ** 60), (2.0 ** -80, 2.0 ** 80)):
        scales = torch.full((64,), of_w, device=DEV)
        s[0, 0, :64] = scales
        exact, bound = plain.product(x * of_x, codes[0, 0], scales)
        assert 2.0 ** -125 < exact.abs().min() and exact.abs().max() < 2.0 ** 127
        plain.agree(linear(x * of_x, w, s, 64), exact, bound, (of_x, of_w))


def test_places_that_are_refused():
    gen = generator(7)
    x = rows_of(gen, 20, 128)
    _, _, w, s = plain.random_weight(gen, 1, 1, 128, 128, DEV)
    with pytest.raises(ops.KernelError, match="lie on the rows"):
        ops.linear_8bit(x, w, s, x)
    flat = rows_of(gen, 64, 128, F32).reshape(-1)
    with pytest.raises(ops.KernelError, match="lie on the rows"):
        ops.linear_8bit(flat[:2560].view(20, 128), w, s, flat[2000:4560].view(20, 128))
    odd = torch.zeros(1 << 16, dtype=torch.uint8, device=DEV)[1:]
    with pytest.raises(ops.KernelError, match="scratch starts on 16 bytes"):
        linear(x, w, s, 128, scratch=odd)
    _, _, w_in, s_in = plain.random_weight(gen, 1, 2, 64, 128, DEV)
    _, _, w_down, s_down = plain.random_weight(gen, 1, 1, 128, 64, DEV)
    for rows in (1, 20):
        with pytest.raises(ops.KernelError, match="scratch starts on 16 bytes"):
            ops.gated_8bit(x[:rows], w_in, s_in, w_down, s_down, torch.empty((rows, 128), device=DEV), width=64, scratch=odd)
    room = torch.zeros(w.numel() + 64, dtype=torch.int8, device=DEV)
    with pytest.raises(ops.KernelError, match="start on 16 bytes"):
        linear(x, room[1:1 + w.numel()].view(w.shape), s, 128)
    for wrong in (x.to(torch.float16), x.to(torch.float64)):
        with pytest.raises(ops.KernelError, match="float32 and bfloat16"):
            linear(wrong, w, s, 128)
    with pytest.raises(ops.KernelError, match="not contiguous"):
        linear(rows_of(gen, 128, 20).t(), *plain.random_weight(gen, 1, 1, 128, 128, DEV)[2:], 128)
    torch.cuda.synchronize()


def test_no_rows():
    _, _, w, s = plain.random_weight(generator(), 1, 1, 40, 100, DEV)
    ops.linear_8bit(torch.zeros((0, 100), device=DEV), w, s, torch.zeros((0, 40), device=DEV))
    _, _, w_in, s_in = plain.random_weight(generator(), 1, 2, 40, 100, DEV)
    _, _, w_down, s_down = plain.random_weight(generator(), 1, 1, 100, 40, DEV)
    ops.gated_8bit(torch.zeros((0, 100), device=DEV), w_in, s_in, w_down, s_down, torch.zeros((0, 100), device=DEV), width=40)
    ops.experts_8bit(torch.zeros((0, 100), device=DEV), torch.zeros((0, 2), dtype=torch.int32, device=DEV), torch.zeros((0, 2), device=DEV), w_in, s_in, w_down, s_down,
                     torch.zeros((0, 100), device=DEV), width=40)


def test_scratch_of_ones_own():
    gen = generator(6)
    x = rows_of(gen, 50, 100)
    _, _, w, s = plain.random_weight(gen, 1, 1, 40, 100, DEV)
    scratch = torch.full((ops.linear_8bit_scratch(50, 100) + 512,), 77, dtype=torch.uint8, device=DEV)
    assert torch.equal(linear(x, w, s, 40, scratch=scratch[:-512]), linear(x, w, s, 40))
    assert (scratch[-512:] == 77).all()
    with pytest.raises(ops.KernelError, match="are needed"):
        linear(x, w, s, 40, scratch=scratch[:1024])


# ------------------------------------------------------------------------------------------------ a gated block

def gated_weights(gen, experts, inner, width):
    return plain.random_weight(gen, experts, 2, width, inner, DEV), plain.random_weight(gen, experts, 1, inner, width, DEV)


@pytest.mark.parametrize("activation, limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("silu", 1.5)])
@pytest.mark.parametrize("rows, inner, width", [(1, 128, 16), (3, 100, 33), (40, 300, 129), (128, 256, 2048), (129, 1000, 257), (500, 512, 640), (1, 2048, 8192), (700, 1536, 4000)])
def test_gated(rows, inner, width, activation, limit):
    gen = generator(rows + width)
    dtype, result = ((BF16, F32), (F32, BF16))[rows % 2]
    x = rows_of(gen, rows, inner, dtype)
    (ic, iscale, w_in, s_in), (dc, dscale, w_down, s_down) = gated_weights(gen, 1, inner, width)
    out = torch.full((rows, inner), float("nan"), dtype=result, device=DEV)
    ops.gated_8bit(x, w_in, s_in, w_down, s_down, out, width=width, activation=activation, gate_limit=limit)
    exact, bound = plain.block(x, ic[0], iscale[0], dc[0, 0], dscale[0, 0], activation, limit)
    plain.agree(out, exact, bound)


def test_gates_far_out():
    # gates of -200 .. 200: silu is 0 there or its argument, and never a NaN
    x = torch.ones((2, 128), device=DEV)
    codes = torch.zeros((1, 2, 5, 128), device=DEV, dtype=torch.float64)
    codes[0, 0] = torch.tensor([-127.0, -20.0, 0.0, 20.0, 127.0], device=DEV)[:, None]
    codes[0, 1] = 127
    scales = torch.full((1, 2, 5), 200 / 127 / 128, device=DEV)
    w_in, s_in = plain.laid_out(codes, scales)
    dc, dscale, w_down, s_down = plain.random_weight(generator(), 1, 1, 128, 5, DEV)
    for activation in ("silu", "gelu_tanh"):
        out = torch.empty((2, 128), device=DEV)
        ops.gated_8bit(x, w_in, s_in, w_down, s_down, out, width=5, activation=activation)
        exact, bound = plain.block(x, codes[0], scales[0], dc[0, 0], dscale[0, 0], activation)
        plain.agree(out, exact, bound)


# ------------------------------------------------------------------------------------------------ routed experts

def experts_case(gen, tokens, inner, width, experts, top_k, dtype=BF16, like=None):
    x = rows_of(gen, tokens, inner, dtype)
    liking = torch.randn((tokens, experts), generator=gen, device=DEV) + (0 if like is None else like)
    top, ids = liking.topk(top_k, -1)
    return x, ids.to(torch.int32), torch.softmax(top, -1), gated_weights(gen, experts, inner, width)


def check_experts(x, ids, weights, parts, limit=0.0, dtype=F32):
    (ic, iscale, w_in, s_in), (dc, dscale, w_down, s_down) = parts
    width = ic.shape[2]
    out = torch.full(x.shape, float("nan"), dtype=dtype, device=DEV)
    ops.experts_8bit(x, ids, weights, w_in, s_in, w_down, s_down, out, width=width, gate_limit=limit)
    exact, bound = torch.zeros(x.shape, dtype=torch.float64, device=DEV), torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(exact)
    for e in range(ic.shape[0]):
        token, rank = torch.nonzero(ids == e, as_tuple=True)
        if token.numel():
            y, off = plain.block(x[token], ic[e], iscale[e], dc[e, 0], dscale[e, 0], "silu", limit)
            weight = weights[token, rank].double()[:, None]
            exact.index_add_(0, token, y * weight)
            bound.index_add_(0, token, off * weight.abs())
            size.index_add_(0, token, y.abs() * weight.abs())
    plain.agree(out, exact, bound + (ids.shape[1] + 1) * plain.U * size)            # a product and a sum a rank
    return out


@pytest.mark.parametrize("tokens, inner, width, experts, top_k, limit", [
    (1, 128, 16, 4, 1, 0.0), (1, 256, 128, 64, 8, 0.0), (3, 100, 33, 5, 5, 1.5), (17, 300, 129, 20, 3, 0.0), (64, 512, 256, 8, 2, 0.0), (130, 1000, 504, 20, 3, 7.0),
    (500, 256, 384, 4, 2, 0.0), (1500, 384, 256, 3, 1, 0.0), (2000, 256, 128, 300, 8, 0.0), (7, 128, 64, 1100, 4, 0.0)])
def test_experts(tokens, inner, width, experts, top_k, limit):
    gen = generator(tokens + width)
    check_experts(*experts_case(gen, tokens, inner, width, experts, top_k, (BF16, F32)[tokens % 2]), limit, (F32, BF16)[tokens % 2])


def test_experts_that_nearly_all_tokens_pick():
    gen = generator(8)
    like = torch.zeros(40, device=DEV)
    like[17] = 9.0
    check_experts(*experts_case(gen, 900, 256, 128, 40, 2, like=like))


def test_ids_that_name_no_expert_and_experts_named_twice():
    gen = generator(9)
    x, ids, weights, parts = experts_case(gen, 60, 256, 96, 6, 3)
    ids[3] = -1
    ids[4, 1] = -1
    ids[5, 0] = 6
    ids[6, 2] = 1 << 30
    ids[7] = 2                                       # one expert three times
    out = check_experts(x, ids, weights, parts)
    assert not out[3].any()
    ids[:] = -1
    assert not check_experts(x, ids, weights, parts).any()


def test_experts_with_lists_of_the_frameworks_own():
    """The products over the lists that a router's step makes, as the routed experts of a model call them."""
    gen = generator(10)
    x, ids, weights, parts = experts_case(gen, 300, 256, 128, 12, 4)
    (_, _, w_in, s_in), (_, _, w_down, s_down) = parts
    want = torch.empty((300, 256), device=DEV)
    ops.experts_8bit(x, ids, weights, w_in, s_in, w_down, s_down, want, width=128)
    for tile_rows in ops.EXPERT_TILES_8BIT:
        n, most = ids.numel(), ids.numel() // tile_rows + 12
        new = lambda count: torch.zeros(count, dtype=torch.int32, device=DEV)
        counts, offsets, sorted_token, row_of_assign, tile_expert, tile_row0, num_tiles = new((n + 1023) // 1024 * 12), new(13), new(n), new(n), new(most), new(most), new(1)
        ops.expert_plan(ids, 12, tile_rows, counts, offsets, sorted_token, row_of_assign, tile_expert, tile_row0, num_tiles)
        y = torch.full((n, 256), float("nan"), device=DEV)
        ops.expert_rows_8bit(x, row_of_assign, (tile_expert, tile_row0, num_tiles, offsets), most, tile_rows, w_in, s_in, w_down, s_down, y, width=128)
        out = torch.empty((300, 256), device=DEV)
        ops.expert_combine(y, weights, row_of_assign, out)
        assert torch.equal(out, want), tile_rows


def test_lists_that_point_out_of_place_reach_nothing_outside():
    gen = generator(13)
    x, _, _, parts = experts_case(gen, 24, 256, 128, 3, 1)
    (ic, iscale, w_in, s_in), (dc, dscale, w_down, s_down) = parts
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    room = torch.full((24 * 256 + 512,), 5.0, device=DEV)
    y = room[256:256 + 24 * 256].view(24, 256)
    order = torch.arange(24, dtype=torch.int32, device=DEV)
    order[5], order[6] = -1, 1 << 20
    # tiles of experts 0 .. 2 in their places, then ones of no expert and of no rows; more of them than the lists hold
    lists = (ints(0, 1, 2, 99, -7, 1), ints(0, 8, 16, 1 << 20, -100, 1 << 28), ints(1 << 20), ints(0, 8, 16, 24))
    ops.expert_rows_8bit(x, order, lists, 6, 8, w_in, s_in, w_down, s_down, y, width=128)
    torch.cuda.synchronize()
    exact, bound = plain.block(x[8:16], ic[1], iscale[1], dc[1, 0], dscale[1, 0])
    plain.agree(y[8:16], exact, bound)
    assert (room[:256] == 5).all() and (room[256 + 24 * 256:] == 5).all()


# ------------------------------------------------------------------------------------------------ streams and graphs

def test_on_another_stream_and_recorded():
    gen = generator(11)
    x, ids, weights, parts = experts_case(gen, 20, 256, 128, 12, 4)
    (_, _, w_in, s_in), (_, _, w_down, s_down) = parts
    _, _, w, s = plain.random_weight(gen, 1, 1, 300, 256, DEV)
    inputs = [rows_of(gen, 20, 256) for _ in range(3)]

    def calls(outs):
        ops.linear_8bit(x, w, s, outs[0])
        ops.gated_8bit(x, w_in[:1], s_in[:1], w_down[:1], s_down[:1], outs[1], width=128)
        ops.experts_8bit(x, ids, weights, w_in, s_in, w_down, s_down, outs[2], width=128)

    def new():
        return [torch.zeros((20, n), device=DEV) for n in (300, 256, 256)]
    wants = []
    for data in inputs:
        x.copy_(data)
        outs = new()
        calls(outs)
        wants.append(outs)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = new()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        calls(outs)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, wants[2]))
    graphs = []
    for _ in range(2):
        outs, graph = new(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            calls(outs)
        graphs.append((graph, outs))
    for data, want in zip(inputs, wants):
        x.copy_(data)
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_weights_written_right_before_a_call():
    """The product asks for its weights ahead of the end of the kernel that makes the tokens' codes: what wrote the weights before it has ended by then."""
    gen = generator(12)
    x = rows_of(gen, 2, 4096)
    weights = [plain.random_weight(gen, 1, 1, 4096, 4096, DEV)[2:] for _ in range(2)]
    wants = [linear(x, w, s, 4096) for w, s in weights]
    w, s = torch.zeros_like(weights[0][0]), torch.zeros_like(weights[0][1])
    for turn in range(20):
        w.copy_(weights[turn % 2][0])
        s.copy_(weights[turn % 2][1])
        assert torch.equal(linear(x, w, s, 4096), wants[turn % 2])
