"""Products in 8-bit integers on the device at the ends of their sizes, and two of them at once."""
import pytest
import torch

import plain_products_8bit as plain
from fieldrun_b200.csrc import ops
from test_products_8bit_gpu import check_experts, experts_case, gated_weights, generator, rows_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    torch.cuda.synchronize()
    ops.tc_status_check(torch.device("cuda:0"))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens, inner, width, experts, top_k", [
    (2100, 128, 64, 40, 8),             # more assignments than the lists' kernel keeps in registers, by less than a round of its threads
    (9000, 128, 32, 7, 3), (3, 256, 32, 200, 128), (1, 128, 16, 8192, 5), (300, 1, 1, 4, 2), (5, 129, 1, 3, 3)])
def test_experts_at_the_ends(tokens, inner, width, experts, top_k):
    gen = generator(tokens)
    check_experts(*experts_case(gen, tokens, inner, width, experts, top_k), dtype=F32)


@pytest.mark.parametrize("rows", [1, 9, 300])
@pytest.mark.parametrize("inner, width", [(1, 1), (1, 700), (700, 1), (127, 129)])
def test_gated_at_the_ends(rows, inner, width):
    gen = generator(rows + width)
    x = rows_of(gen, rows, inner)
    (ic, iscale, w_in, s_in), (dc, dscale, w_down, s_down) = gated_weights(gen, 1, inner, width)
    out = torch.full((rows, inner), float("nan"), device=DEV)
    ops.gated_8bit(x, w_in, s_in, w_down, s_down, out, width=width)
    plain.agree(out, *plain.block(x, ic[0], iscale[0], dc[0, 0], dscale[0, 0]))


def test_a_middle_beyond_32_bits_of_places():
    gen, rows, inner, width = generator(4), 70_001, 128, 31_000
    x = rows_of(gen, rows, inner)
    (ic, iscale, w_in, s_in), (dc, dscale, w_down, s_down) = gated_weights(gen, 1, inner, width)
    out = torch.empty((rows, inner), device=DEV)
    ops.gated_8bit(x, w_in, s_in, w_down, s_down, out, width=width)
    for some in (slice(0, 100), slice(69_270, 69_320), slice(rows - 100, rows)):
        plain.agree(out[some], *plain.block(x[some], ic[0], iscale[0], dc[0, 0], dscale[0, 0]))


@pytest.mark.parametrize("inner", [8, 600])
def test_more_rows_than_a_grid_has_blocks(inner):
    rows = (1 << 22) + 5 if inner == 8 else (1 << 21) + 3
    x = torch.randn((rows, inner), generator=generator(5), device=DEV).to(BF16)
    codes, scales = torch.full((rows, plain.up(inner, 128)), 99, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    ops.rows_8bit(x, codes, scales)
    for some in (slice(0, 1000), slice(rows // 2 - 500, rows // 2 + 500), slice(rows - 1000, rows)):
        want, step = plain.codes_of(x[some])
        assert torch.equal(codes[some, :inner].double(), want) and not codes[some, inner:].any()
        assert ((scales[some].double() - step[:, 0]).abs() <= plain.U * step[:, 0]).all()


def test_two_streams_at_once():
    """Calls of every form side by side, whose blocks share SMs and their tensor memory."""
    gen = generator(6)
    _, _, w, s = plain.random_weight(gen, 1, 1, 2000, 512, DEV)
    (_, _, w_in, s_in), (_, _, w_down, s_down) = gated_weights(gen, 4, 512, 256)
    xs = [rows_of(gen, rows, 512) for rows in (1, 20, 400)]
    ids = [torch.randint(0, 4, (x.shape[0], 2), generator=gen, device=DEV, dtype=torch.int32) for x in xs]
    shares = [torch.rand((x.shape[0], 2), generator=gen, device=DEV) for x in xs]

    def calls(order):
        outs = {}
        for n in order:
            x = xs[n]
            outs[n] = [torch.empty((x.shape[0], f), device=DEV) for f in (2000, 512, 512)]
            ops.linear_8bit(x, w, s, outs[n][0])
            ops.gated_8bit(x, w_in[:1], s_in[:1], w_down[:1], s_down[:1], outs[n][1], width=256)
            ops.experts_8bit(x, ids[n], shares[n], w_in, s_in, w_down, s_down, outs[n][2], width=256)
        return outs
    want = calls((0, 1, 2))
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    torch.cuda.synchronize()
    for turn in range(15):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(calls([(k + turn + i) % 3 for i in range(3)]))
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for n in want for a, b in zip(outs[n], want[n]))
