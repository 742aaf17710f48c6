"""Models whose weights are held in 8 bits: every product of every step against 64 bits, the same steps recorded and cut in other ways, the
entry points that make such a model."""
import importlib
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import fieldrun_b200 as fr
import plain_products_8bit as plain
from fieldrun_b200.csrc import ops
from fieldrun_b200.parts.feed_forward import RoutedExperts
from fieldrun_b200.parts.linear import Weight8

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MODELS = [("tiny", "a"), ("tiny", "b"), ("tiny", "d"), ("bamasun", "C"), ("fotanex", "C"), ("depelix", "C"), ("bakasun", "A"), ("bakasun", "C"), ("duzinex", "C"),
          ("kifunex", "B"), ("kifunex", "C")]


def model(design, name, weight_dtype="int8", **more):
    config, init = importlib.import_module(f"{design}_configs").ALL[name]
    return fr.random_model(config, init, weight_dtype=weight_dtype, **{"max_tokens": 4096, "num_slots": 6, **more}), config


def vocabulary(config):
    return config.get("vocab_size") or config["vocab"]


@pytest.fixture
def watched(monkeypatch):
    """Compares every product in 8 bits with 64 bits over the same rows, codes and scales."""
    seen = []

    def linear(x, codes, scales, out, **more):
        inner(x, codes, scales, out, **more)
        f, k = out.shape[1], x.shape[1]
        plain.agree(out, *plain.product(x, codes[0, 0, :f, :k], scales[0, 0, :f]), "linear")
        seen.append("linear")

    def gated(x, ic, iscale, dc, dscale, out, *, width, activation="silu", **more):
        inner_gated(x, ic, iscale, dc, dscale, out, width=width, activation=activation, **more)
        d = x.shape[1]
        plain.agree(out, *plain.block(x, ic[0, :, :width, :d], iscale[0, :, :width], dc[0, 0, :d, :width], dscale[0, 0, :d], activation), "gated")
        seen.append("gated")

    def experts(x, row_of_assign, lists, max_tiles, tile_rows, ic, iscale, dc, dscale, y, *, width, gate_limit=0.0, **more):
        inner_experts(x, row_of_assign, lists, max_tiles, tile_rows, ic, iscale, dc, dscale, y, width=width, gate_limit=gate_limit, **more)
        d, offsets = x.shape[1], lists[3].tolist()
        rows = x
        if row_of_assign is not None:
            rows = torch.empty((y.shape[0], d), dtype=x.dtype, device=x.device)
            rows[row_of_assign.reshape(-1).long()] = x.repeat_interleave(y.shape[0] // x.shape[0], 0)
        assert offsets[-1] == y.shape[0]
        for e, (first, end) in enumerate(zip(offsets, offsets[1:])):
            if end > first:
                plain.agree(y[first:end], *plain.block(rows[first:end], ic[e, :, :width, :d], iscale[e, :, :width], dc[e, 0, :d, :width], dscale[e, 0, :d], "silu",
                                                       gate_limit), "experts")
        seen.append("experts")
    inner, inner_gated, inner_experts = ops.linear_8bit, ops.gated_8bit, ops.expert_rows_8bit
    monkeypatch.setattr(ops, "linear_8bit", linear)
    monkeypatch.setattr(ops, "gated_8bit", gated)
    monkeypatch.setattr(ops, "expert_rows_8bit", experts)
    return seen


@pytest.mark.parametrize("design,name", MODELS)
def test_every_product_of_a_model(design, name, watched):
    lm, config = model(design, name)
    engine = lm.engine
    engine.record_steps = False
    rng = np.random.default_rng(3)
    draw = lambda n: rng.integers(0, vocabulary(config), size=n).tolist()
    slots = [engine.new_sequence() for _ in range(4)]
    out = [engine.step(slots, [draw(n) for n in (70, 9, 200, 1)])]        # prompts
    out.append(engine.step(slots, [draw(1) for _ in slots]))               # single tokens
    out.append(engine.step(slots[:1], [draw(1)]))
    out.append(engine.step(slots[1:], [draw(130), draw(66), draw(64)]))    # prompts that go on
    engine.check()
    assert all(torch.isfinite(o).all() for o in out) and watched


@pytest.mark.parametrize("design,name", MODELS)
def test_a_recorded_step_gives_what_a_direct_one_gives(design, name):
    lm, config = model(design, name)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, vocabulary(config), size=n).tolist() for n in (40, 3, 130)]
    logits = {}
    for recorded in (True, False):
        engine = lm.engine
        engine.record_steps = recorded
        slots = [engine.new_sequence() for _ in prompts]
        out = [engine.step(slots, prompts)]
        for step in range(4):                        # the recording is made at the first, replayed for the others
            out.append(engine.step(slots, [[(7 * step + i) % vocabulary(config)] for i in range(3)]))
        engine.check()
        logits[recorded] = torch.cat(out).cpu()
        for s in slots:
            engine.release(s)
    assert lm.engine.steps_replayed >= 3 or not lm.model.replayable
    assert torch.isfinite(logits[True]).all() and torch.equal(logits[True], logits[False])


def test_weights_are_the_models_rounded_row_by_row():
    (lm, _), (whole, _) = model("tiny", "d"), model("tiny", "d", None)
    checked = 0

    def same(weight, matrices, expert=0):
        nonlocal checked
        for part, matrix in enumerate(matrices):
            codes, step = plain.codes_of(matrix)
            f, k = matrix.shape
            assert torch.equal(weight.codes[expert, part, :f, :k].double(), codes)
            assert ((weight.scales[expert, part, :f].double() - step[:, 0]).abs() <= plain.U * step[:, 0]).all()
            checked += 1
    for block, other in zip(lm.model.blocks, whole.model.blocks):
        same(block.mixer.w_qkv, [other.mixer.w_qkv])
        same(block.mixer.w_o, [other.mixer.w_o])
        mlp, plain_mlp = block.feed_forward, other.feed_forward
        assert isinstance(mlp, RoutedExperts) and mlp.router.dtype == torch.float32
        for e in range(mlp.num_experts):
            same(mlp.w13, plain_mlp.w13[e].view(2, mlp.expert_width, -1), e)
            same(mlp.w2, [plain_mlp.w2[e]], e)
    assert checked
    # what the model counts: a byte an entry and four a channel where sizes need no filling, and half of what two bytes an entry take at most
    held = lambda m: sum(t.numel() * t.element_size() for part in m.all_parts() for w in vars(part).values() if isinstance(w, Weight8) for t in w.pair)
    assert held(lm.model) > 0 and lm.model.weight_bytes() < whole.model.weight_bytes()


def test_generation():
    lm, _ = model("tiny", "d", cache_dtype="int8")
    prompts = [[5, 17, 3], [9], list(range(100))]
    out = lm.generate_batch(prompts, 20, eos=[])
    assert [len(o) for o in out] == [20, 20, 20] and out == lm.generate_batch(prompts, 20, eos=[])
    assert lm.generate(prompts[2], 20) == lm.generate(prompts[2], 20)
    assert lm.logits(prompts[2]).isfinite().all()


def test_command_line_and_replay(tmp_path):
    from tiny_configs import CONFIG_B, INIT_B
    folder = str(tmp_path / "model")
    fr.write_random_model(folder, CONFIG_B, INIT_B)
    ids = tmp_path / "ids.json"
    ids.write_text(json.dumps({"holdout_ids": list(range(30))}))
    run = lambda *args, **more: subprocess.run([sys.executable, *args], cwd=ROOT, capture_output=True, text=True, timeout=600, **more)
    want = fr.load(folder, max_tokens=64, weight_dtype="int8").generate(list(range(12)), 6)
    proc = run("-m", "fieldrun_b200", "--model", folder, "--ids", str(ids), "--ctx", "12", "--generate", "6", "--eos", "none", "--weight-dtype", "int8")
    assert proc.returncode == 0, proc.stderr[-2000:]
    assert " ".join(map(str, want)) in proc.stdout
    proc = run("-m", "fieldrun_b200", "--model", folder, "--ids", str(ids), "--ctx", "12", "--generate", "6", "--dtype", "float32", "--weight-dtype", "int8")
    assert proc.returncode == 1 and "for bfloat16 models" in proc.stderr
    out = str(tmp_path / "out")
    step = {"step": 0, "entries": [{"id": "a", "tokens": list(range(12)), "want": [11]}], "end": []}
    proc = run(os.path.join(ROOT, "bin", "trace_run"), "--model", folder, "--dtype", "bfloat16", "--out", out, "--max-tokens", "64", "--weight-dtype", "int8",
               input=json.dumps(step) + "\n")
    assert proc.returncode == 0, proc.stderr[-2000:]
    logits = np.fromfile(os.path.join(out, "0.f32"), dtype="<f4")
    assert int(logits.argmax()) == want[0]
