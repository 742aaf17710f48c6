"""Codes of rows on the device, bit for bit, as both of the kernels that round make them: the rows' own, and the product of up to eight tokens."""
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


def generator(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def codes_by_rows(x):
    codes, scales = torch.full((x.shape[0], plain.up(x.shape[1], 128)), 99, dtype=torch.int8, device=DEV), torch.empty(x.shape[0], device=DEV)
    ops.rows_8bit(x, codes, scales)
    return codes[:, :x.shape[1]].double()


def codes_by_product(x):
    """A weight of ones on its diagonal: every result is its token's scale times one code, off by a rounding."""
    inner = x.shape[1]
    w, s = torch.zeros(ops.weight_8bit_shape(1, 1, inner, inner), dtype=torch.int8, device=DEV), torch.ones((1, 1, plain.up(inner, 16)), device=DEV)
    w[0, 0].fill_diagonal_(1)
    out = torch.empty((x.shape[0], inner), device=DEV)
    ops.linear_8bit(x, w, s, out)
    _, step = plain.codes_of(x)
    return torch.round(out.double() / step.clamp_min(1e-300))


def next_to_middles(gen, rows, inner):
    """float32 entries up to two places off the middle of two codes."""
    top = torch.rand((rows, 1), generator=gen, device=DEV) + 1
    half = torch.randint(-126, 126, (rows, inner), generator=gen, device=DEV).double() + 0.5
    x = (half * top.double() / 127).float()
    x = (x.view(torch.int32) + torch.randint(-2, 3, (rows, inner), generator=gen, device=DEV, dtype=torch.int32)).view(torch.float32).clone()
    x[:, 0] = top[:, 0]
    return x


@pytest.mark.parametrize("rows, inner", [(1, 8192), (2, 4096), (3, 2500), (4, 4096), (5, 2048), (8, 2047), (9, 2048), (300, 1000)])
def test_float32_entries_next_to_middles(rows, inner):
    gen = generator(rows)
    for _ in range(4):
        x = next_to_middles(gen, rows, inner)
        want, _ = plain.codes_of(x)
        assert torch.equal(codes_by_rows(x), want) and torch.equal(codes_by_product(x), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_rows_results_are_its_own_however_it_was_rounded(dtype):
    """One to eight rows are rounded by the product, more by a kernel of their own; entries lie next to middles."""
    gen = generator(7)
    x = next_to_middles(gen, 300, 1500).to(dtype)
    _, _, w, s = plain.random_weight(gen, 1, 1, 700, 1500, DEV)
    whole = torch.empty((300, 700), device=DEV)
    ops.linear_8bit(x, w, s, whole)
    for first, count in [(0, 1), (5, 2), (9, 3), (100, 5), (250, 8), (291, 9), (17, 130)]:
        out = torch.empty((count, 700), device=DEV)
        ops.linear_8bit(x[first:first + count], w, s, out)
        assert torch.equal(out, whole[first:first + count]), (first, count)


def test_every_pair_of_bfloat16_significands():
    """Row a has the largest entry a = 128 .. 255 and every entry of eight bits, halved up to eight times, that is at most a."""
    x = torch.arange(128, 256, device=DEV)[None, :] * torch.exp2(-torch.arange(9.0, device=DEV))[:, None]
    x = torch.cat([x.reshape(-1), torch.zeros(2048 - x.numel(), device=DEV)]).expand(128, -1)
    a = torch.arange(128.0, 256.0, device=DEV)[:, None]
    x = torch.where(x <= a, x, a)
    x[:, 1::2] *= -1
    for power in (-90, 0, 100):
        rows = (x * 2.0 ** power).to(BF16)
        want, _ = plain.codes_of(rows)
        assert torch.equal(codes_by_rows(rows), want)
        for first in range(0, 128, 8):
            assert torch.equal(codes_by_product(rows[first:first + 8]), want[first:first + 8])


def test_tokens_take_the_same_time_whatever_their_largest_entry():
    """No largest entry sends a bfloat16 token to a slower code: 254 and 255, 8 tokens, the least of several recorded runs, with half as much to spare."""
    gen = generator(3)
    x = torch.randint(-250, 250, (8, 2048), generator=gen, device=DEV).float().to(BF16)
    weights = [plain.random_weight(gen, 1, 1, 6144, 2048, DEV)[2:] for _ in range(4)]
    out, took = torch.empty((8, 6144), device=DEV), {}
    for top in (255, 254):
        x[:, 5] = top
        ops.linear_8bit(x, *weights[0], out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for n in range(40):
                ops.linear_8bit(x, *weights[n % 4], out)
        times = []
        for _ in range(8):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            graph.replay()
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        took[top] = min(times)
    assert took[254] < 1.5 * took[255], took
