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
