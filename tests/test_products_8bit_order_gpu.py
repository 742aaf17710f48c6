"""Products in 8-bit integers on the device right behind the kernels that they start beside: what those still do, and what they have just written."""
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


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def recorded(calls, times=1):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for _ in range(times):
        graph.replay()
    torch.cuda.synchronize()


def prompt_attention(gen, tokens, heads, head_dim):
    """A prompt's attention on the tensor cores: the call, and where its output goes."""
    pages = tokens // 64
    rows = lambda *shape: (0.3 * torch.randn(shape, generator=gen, device=DEV)).to(BF16)
    q, k, v = rows(tokens, heads * head_dim), rows(pages, 1, 64, head_dim), rows(pages, 1, head_dim, 64)
    table, tiles = torch.arange(pages, dtype=torch.int32, device=DEV)[None], torch.arange(0, tokens, 128, dtype=torch.int32, device=DEV)
    of_sequence, zero, length, ends, out = torch.zeros_like(tiles), ints(0), ints(tokens), ints(0, tokens), torch.empty_like(q)
    return lambda: ops.attention_prefill_tc(q, k, v, table, of_sequence, tiles, zero, zero, length, ends, out, num_heads=heads, num_kv_heads=1,
                                            head_dim=head_dim, scale=head_dim ** -0.5, window=None), out


@pytest.mark.parametrize("weights_final", [False, True])
@pytest.mark.parametrize("rows, inner, features", [(1, 128, 16), (4, 256, 2048), (9, 128, 4096), (200, 384, 5000)])
def test_behind_a_kernel_that_holds_tensor_memory(rows, inner, features, weights_final):
    """Both take columns of an SM's tensor memory; the product's blocks are small enough to lie beside the attention's."""
    gen = generator(rows)
    attend, attended = prompt_attention(gen, 1024, 16, 64)
    x = torch.randn((rows, inner), generator=gen, device=DEV).to(BF16)
    codes, scales, w, s = plain.random_weight(gen, 1, 1, features, inner, DEV)
    outs = [torch.empty((rows, features), device=DEV) for _ in range(3)]

    def calls():
        for out in outs:
            attend()
            ops.linear_8bit(x, w, s, out, weights_final=weights_final)
    attend()
    want = attended.clone()
    recorded(calls, 20)
    exact, bound = plain.product(x, codes[0, 0], scales[0, 0])
    for out in outs:
        plain.agree(out, exact, bound)
    assert torch.equal(attended, want)
