"""Products in 8-bit integers on the device right behind the kernels that they start beside: what those still do, and what they have just written."""
import json
import os
import subprocess
import sys

import pytest
import torch

import plain_products_8bit as plain
from fieldrun_b200.csrc import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
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


# Records products of every form and says how many of the recording's kernels start beside the one before them, and what came out.
SWITCHED = """
import ctypes, json, sys
sys.path.insert(0, "tests")
import torch
import plain_products_8bit as plain
from fieldrun_b200.csrc import ops
gen = torch.Generator(device="cuda").manual_seed(1)
weight = lambda *sizes: plain.random_weight(gen, *sizes, "cuda")[2:]
w, w_in, w_down = weight(1, 1, 300, 256), weight(4, 2, 128, 256), weight(4, 1, 256, 128)
xs = [torch.randn((rows, 256), generator=gen, device="cuda") for rows in (2, 20, 300)]
outs = [[torch.empty((len(x), n), device="cuda") for n in (300, 256, 256)] for x in xs]
ids = [torch.randint(0, 4, (len(x), 2), generator=gen, device="cuda", dtype=torch.int32) for x in xs]
shares = [torch.rand((len(x), 2), generator=gen, device="cuda") for x in xs]

def calls():
    for x, out, i, s in zip(xs, outs, ids, shares):
        ops.linear_8bit(x, *w, out[0])
        ops.gated_8bit(x, w_in[0][:1], w_in[1][:1], w_down[0][:1], w_down[1][:1], out[1], width=128)
        ops.experts_8bit(x, i, s, *w_in, *w_down, out[2], width=128)
calls()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph(keep_graph=True)
with torch.cuda.graph(graph):
    calls()
graph.instantiate()
graph.replay()
torch.cuda.synchronize()
ops.tc_status_check("cuda:0")
driver, count = ctypes.CDLL("libcuda.so.1"), ctypes.c_size_t(0)
raw = ctypes.c_void_p(graph.raw_cuda_graph())
assert driver.cuGraphGetEdges_v2(raw, None, None, None, ctypes.byref(count)) == 0
nodes, data = [(ctypes.c_void_p * count.value)() for _ in range(2)], (ctypes.c_ubyte * (8 * count.value))()
assert driver.cuGraphGetEdges_v2(raw, *nodes, data, ctypes.byref(count)) == 0
print(json.dumps({"edges": count.value, "early": sum(kind == 1 for kind in data[2::8]),
                  "outs": [o.double().sum().item().hex() for out in outs for o in out]}))
"""


def test_the_switch_for_early_starts():
    said = {}
    for most in ("", "0"):
        proc = subprocess.run([sys.executable, "-c", SWITCHED], cwd=ROOT, capture_output=True, text=True, timeout=600, env={**os.environ, "FIELDRUN_B200_PDL": most})
        assert proc.returncode == 0, proc.stderr[-2000:]
        said[most] = json.loads(proc.stdout.splitlines()[-1])
    assert said[""]["early"] > 20 and said["0"]["early"] == 0
    assert said[""]["edges"] == said["0"]["edges"] and said[""]["outs"] == said["0"]["outs"]


# ------------------------------------------------------------------------------------------------ what was written right before
#
# Every call here stands in one recording right behind a kernel of the framework that lets the next one start while it still writes, and reads what
# that one writes; from turn to turn that is something else, so that a read that comes too early sees the turn before.

TURNS = 12


def matrix(gen, features, inner):
    return (torch.randn((features, inner), generator=gen, device=DEV) / inner ** 0.5).to(BF16)


def in_turns(write, call, out_shape, choices=2):
    """write(n) then call(out) for n = 0, 1, .. in turn, recorded in one piece, against each by itself."""
    wants = []
    for n in range(choices):
        out = torch.empty(out_shape, device=DEV)
        write(n)
        torch.cuda.synchronize()
        call(out)
        torch.cuda.synchronize()
        wants.append(out)
    assert not any(torch.equal(a, b) for a, b in zip(wants, wants[1:]))
    outs = [torch.full(out_shape, float("nan"), device=DEV) for _ in range(TURNS)]

    def turns():
        for n, out in enumerate(outs):
            write(n % choices)
            call(out)
    recorded(turns, 5)
    for n, out in enumerate(outs):
        assert torch.equal(out, wants[n % choices]), n


@pytest.mark.parametrize("rows", [1, 8, 9, 100, 300])
@pytest.mark.parametrize("features, inner", [(144, 2048), (96, 40000), (1000, 500)])
def test_a_layers_weights_written_right_before(rows, features, inner):
    gen = generator(rows)
    x, choices = torch.randn((rows, inner), generator=gen, device=DEV).to(BF16), [matrix(gen, features, inner) for _ in range(2)]
    w, s = ops.weight_8bit(choices[0])
    in_turns(lambda n: ops.weight_8bit(choices[n], codes=w, scales=s), lambda out: ops.linear_8bit(x, w, s, out), (rows, features))


@pytest.mark.parametrize("rows", [1, 8, 9, 100])
@pytest.mark.parametrize("last", ["down", "gate and up"])
def test_a_blocks_weights_written_right_before(rows, last):
    gen, inner, width = generator(rows), 1024, 4000
    x = torch.randn((rows, inner), generator=gen, device=DEV).to(BF16)
    ins, downs = [[matrix(gen, width, inner) for _ in range(2)] for _ in range(2)], [matrix(gen, inner, width) for _ in range(2)]
    (w_in, s_in), (w_down, s_down) = ops.weight_8bit(*ins[0]), ops.weight_8bit(downs[0])

    def write(n):
        steps = [lambda: ops.weight_8bit(*ins[n], codes=w_in, scales=s_in), lambda: ops.weight_8bit(downs[n], codes=w_down, scales=s_down)]
        for step in steps if last == "down" else steps[::-1]:
            step()
    in_turns(write, lambda out: ops.gated_8bit(x, w_in, s_in, w_down, s_down, out, width=width), (rows, inner))


@pytest.mark.parametrize("tokens", [1, 40, 500])
def test_experts_weights_written_right_before(tokens):
    gen, inner, width, experts = generator(tokens), 512, 384, 6
    x, ids = torch.randn((tokens, inner), generator=gen, device=DEV).to(BF16), torch.randint(0, experts, (tokens, 2), generator=gen, device=DEV, dtype=torch.int32)
    shares = torch.rand((tokens, 2), generator=gen, device=DEV)
    choices = [[(matrix(gen, width, inner), matrix(gen, width, inner), matrix(gen, inner, width)) for _ in range(experts)] for _ in range(2)]
    w_in, s_in = (torch.zeros(ops.weight_8bit_shape(experts, 2, width, inner)[:n], dtype=t, device=DEV) for n, t in ((4, torch.int8), (3, F32)))
    w_down, s_down = (torch.zeros(ops.weight_8bit_shape(experts, 1, inner, width)[:n], dtype=t, device=DEV) for n, t in ((4, torch.int8), (3, F32)))

    def write(n):
        for e, (gate, up, down) in enumerate(choices[n]):
            ops.weight_8bit(gate, up, codes=w_in[e:e + 1], scales=s_in[e:e + 1])
            ops.weight_8bit(down, codes=w_down[e:e + 1], scales=s_down[e:e + 1])
    in_turns(write, lambda out: ops.experts_8bit(x, ids, shares, w_in, s_in, w_down, s_down, out, width=width), (tokens, inner))


@pytest.mark.parametrize("tokens", [1, 16, 30, 700])
def test_lists_made_right_before(tokens):
    gen, inner, width, experts, top_k, tile = generator(tokens), 512, 256, 24, 3, 16
    x = torch.randn((tokens, inner), generator=gen, device=DEV).to(BF16)
    w_in, s_in = plain.random_weight(gen, experts, 2, width, inner, DEV)[2:]
    w_down, s_down = plain.random_weight(gen, experts, 1, inner, width, DEV)[2:]
    picks = [torch.stack([torch.randperm(experts, generator=gen, device=DEV)[:top_k] for _ in range(tokens)]).to(torch.int32) for _ in range(3)]
    n, most = tokens * top_k, tokens * top_k // tile + experts
    new = lambda count: torch.zeros(count, dtype=torch.int32, device=DEV)
    counts, offsets, sorted_token, row_of_assign, tile_expert, tile_row0, num_tiles = new((n + 1023) // 1024 * experts), new(experts + 1), new(n), new(n), new(most), new(most), new(1)
    y, shares = torch.empty((n, inner), device=DEV), torch.rand((tokens, top_k), generator=gen, device=DEV)

    def call(out):
        ops.expert_rows_8bit(x, row_of_assign, (tile_expert, tile_row0, num_tiles, offsets), most, tile, w_in, s_in, w_down, s_down, y, width=width)
        ops.expert_combine(y, shares, row_of_assign, out)
    in_turns(lambda k: ops.expert_plan(picks[k], experts, tile, counts, offsets, sorted_token, row_of_assign, tile_expert, tile_row0, num_tiles), call, (tokens, inner), 3)


@pytest.mark.parametrize("rows", [1, 2, 8, 9, 100, 300])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_made_right_before_a_call_with_weights_that_are_final(rows, dtype):
    """weights_final lets the weights, and nothing else, be read beside the kernel before."""
    gen, inner, features, width = generator(rows), 1000, 777, 2100
    table = torch.randn((50, inner), generator=gen, device=DEV).to(BF16)
    w, s = plain.random_weight(gen, 1, 1, features, inner, DEV)[2:]
    w_in, s_in = plain.random_weight(gen, 1, 2, width, inner, DEV)[2:]
    w_down, s_down = plain.random_weight(gen, 1, 1, inner, width, DEV)[2:]
    tokens = [torch.randint(0, 50, (rows,), generator=gen, device=DEV, dtype=torch.int32) for _ in range(3)]
    stream, act = torch.empty((rows, inner), device=DEV), torch.empty((rows, inner), dtype=BF16, device=DEV)
    x = act if dtype == BF16 else stream
    for final in (False, True):
        in_turns(lambda n: ops.embed_rows(tokens[n], table, stream, act=act), lambda out: ops.linear_8bit(x, w, s, out, weights_final=final), (rows, features), 3)
        in_turns(lambda n: ops.embed_rows(tokens[n], table, stream, act=act),
                 lambda out: ops.gated_8bit(x, w_in, s_in, w_down, s_down, out, width=width, weights_final=final), (rows, inner), 3)
    exact, bound = plain.product(x, w[0, 0, :features, :inner], s[0, 0, :features])
    out = torch.empty((rows, features), device=DEV)
    ops.linear_8bit(x, w, s, out, weights_final=True)
    plain.agree(out, exact, bound)


@pytest.mark.parametrize("rows", [1, 8, 9, 200])
def test_layers_one_behind_another(rows):
    """Rows that the product before still stores, read by the next one with weights that are final."""
    gen, inner = generator(rows), 1280
    weights = [plain.random_weight(gen, 1, 1, inner, inner, DEV)[2:] for _ in range(4)]
    xs = [torch.randn((rows, inner), generator=gen, device=DEV) for _ in range(2)]
    x, middles = torch.empty((rows, inner), device=DEV), [torch.empty((rows, inner), device=DEV) for _ in range(3)]

    def call(out):
        for (w, s), before, after in zip(weights, (x, *middles), (*middles, out)):
            ops.linear_8bit(before, w, s, after, weights_final=True)
    in_turns(lambda n: x.copy_(xs[n]), call, (rows, inner))
    want = xs[(TURNS - 1) % 2]
    for w, s in weights:
        after = torch.empty_like(want)
        torch.cuda.synchronize()
        ops.linear_8bit(want, w, s, after)
        torch.cuda.synchronize()
        want = after
    out = torch.empty_like(want)
    call(out)
    assert torch.equal(out, want)
