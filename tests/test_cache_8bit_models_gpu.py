"""Models whose keys and values are held in 8 bits: what every attention of every step gives, against plain float64 over the rows
that the cache holds; the same requests cut into steps in other ways; the entry points that make such a model."""
import importlib
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import cache_8bit_plain as plain
import fieldrun_b200 as fr
from fieldrun_b200.csrc import ops
from fieldrun_b200.parts.attention import GQAAttention

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 64
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MODELS = [("tiny", "b"), ("tiny", "d"), ("bamasun", "C"), ("fotanex", "C"), ("bakasun", "C"), ("duzinex", "C"), ("kifunex", "C")]


def model(design, name, cache_dtype, **more):
    config, init = importlib.import_module(f"{design}_configs").ALL[name]
    return fr.random_model(config, init, cache_dtype=cache_dtype, **{"max_tokens": 4096, "num_slots": 6, **more}), config


def vocabulary(config):
    return config.get("vocab_size") or config["vocab"]


class Watched:
    """Compares every attention of the steps run inside with float64 over the rows of the cache (codes times scales; for prompts rounded to
    bfloat16, as they are read back)."""

    def __init__(self, monkeypatch):
        self.seen = []
        inner = GQAAttention.attend

        def attend(part, ctx, q, line, out, gate=None):
            inner(part, ctx, q, line, out, gate)
            assert line.key_scales is not None and line.keys.dtype in ops.CACHE_8BIT_TYPES
            self.check(part, ctx, q, line, out, gate)
        monkeypatch.setattr(GQAAttention, "attend", attend)

    def rows(self, line, codes, scales, slot, length, rounded):
        pages = line.page_table[slot, :-(-length // PAGE)].long()
        held = (pages >= 0)[:, None, None, None]
        x = codes.view(torch.uint8)[pages.clamp_min(0)].view(codes.dtype).float() * scales[pages.clamp_min(0)][..., None]
        if rounded:
            x = x.to(torch.bfloat16)
        x = torch.where(held, x.double(), torch.full_like(x, float("nan"), dtype=torch.float64)).cpu().numpy()      # pages given back are not looked at
        return x.transpose(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[-1])[:, :length]

    def check(self, part, ctx, q, line, out, gate):
        q = q.double().cpu().numpy().reshape(-1, part.q_heads, part.head_dim)
        got = out.double().cpu().numpy().reshape(-1, part.num_heads, part.value_dim)
        gates = 1 / (1 + np.exp(-gate.double().cpu().numpy())) if gate is not None else None
        slopes = part.slopes.double().cpu().numpy() if part.slopes is not None else None
        sinks = part.sinks.double().cpu().numpy() if part.sinks is not None else None
        group = part.q_heads // part.k_heads
        prompt = not ctx.is_decode
        at = 0
        for slot, start, n in zip(ctx.seq_slots, ctx.seq_starts, ctx.seq_q_lens):
            k = self.rows(line, line.keys, line.key_scales, slot, start + n, prompt)
            v = self.rows(line, line.values, line.value_scales, slot, start + n, prompt)
            places = range(n) if n <= 12 else sorted({0, 1, n // 3, n // 2, n - 2, n - 1})
            for place in places:
                pos = start + place
                want, size, top, reach, span = plain.attend(q[at + place], k, v, pos, scale=part.softmax_scale, group=group, maps=part.maps,
                                                      window=int(part.window) if part.window else None, chunk=part.chunk, keep_first=part.keep_first,
                                                      slopes=slopes, sinks=sinks, softcap=part.softcap)
                # prompts: weights in bfloat16 (2^-8); the softmax's sum is of the unrounded ones
                want, bound = plain.output_bound(want, size, top, reach, span, pos, dim=part.head_dim, codes=None if prompt else line.keys.dtype, group=part.num_heads // part.num_kv_heads,
                                                 maps=part.maps, softcap=part.softcap, slopes=slopes, rounding=2.0 ** -8 if prompt else 2.0 ** -11,
                                                 **(dict(lam=float(part.lam.double()), eps=part.diff_eps, factor=1 - part.diff) if part.maps == 2 else {}))
                if gates is not None:
                    g = gates[at + place][:part.num_heads, None]
                    want, bound = want * g, bound * g + 2.0 ** -8 * np.abs(want * g) * 1.01
                off = np.abs(got[at + place] - want)
                assert (off <= bound).all(), (part.spec.kind, pos, prompt, float((off / bound).max()))
                self.seen.append((prompt, part.head_dim, part.window, part.chunk))
            at += n


@pytest.mark.parametrize("cache_dtype", ["int8", "float8_e4m3fn"])
@pytest.mark.parametrize("design,name", MODELS)
def test_every_attention_of_a_model(design, name, cache_dtype, monkeypatch):
    lm, config = model(design, name, cache_dtype)
    engine = lm.engine
    engine.record_steps = False
    watched = Watched(monkeypatch)
    rng = np.random.default_rng(3)
    draw = lambda n: rng.integers(0, vocabulary(config), size=n).tolist()
    slots = [engine.new_sequence() for _ in range(4)]
    engine.step(slots, [draw(n) for n in (70, 9, 200, 1)])           # prompts
    engine.step(slots, [draw(1) for _ in slots])                     # single tokens
    engine.step(slots[:2], [draw(5), draw(3)])                       # a few tokens more each
    engine.step(slots[1:], [draw(130), draw(66), draw(64)])          # prompts that go on
    engine.step(slots, [draw(1) for _ in slots])
    engine.check()
    assert {p for p, *_ in watched.seen} == {True, False}


@pytest.mark.parametrize("cache_dtype", ["int8", "float8_e4m3fn"])
@pytest.mark.parametrize("design,name", MODELS)
def test_a_recorded_step_gives_what_a_direct_one_gives(design, name, cache_dtype):
    lm, config = model(design, name, cache_dtype)
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
    assert lm.engine.steps_replayed >= 3
    assert torch.isfinite(logits[True]).all() and torch.equal(logits[True], logits[False])


def test_a_sequence_does_not_depend_on_what_ran_in_its_pages_before():
    lm, config = model("tiny", "d", "int8", max_tokens=512, num_slots=2)
    ids = np.random.default_rng(1).integers(0, 300, size=90).tolist()
    first = lm.logits(ids)
    for codes in lm.engine.cache.groups:                             # whatever lies in the pages that the next sequence gets
        codes.key_scales.fill_(float("nan"))
        codes.value_scales.fill_(float("inf"))
        codes.keys.view(torch.uint8).fill_(0x7f)
        codes.values.view(torch.uint8).fill_(0xff)
    assert torch.equal(lm.logits(ids), first)
    slot = lm.engine.new_sequence()
    lm.engine.step([slot], [ids[:70]])
    tail = torch.cat([lm.engine.step([slot], [[t]]) for t in ids[70:]])
    assert torch.isfinite(tail).all()
    # the same rows are attended over, by other kernels: the weights' rounding (2^-8 and 2^-11) and the activations', layer by layer
    assert (tail - first[70:]).abs().max() <= 2.5e-2 * 4 * first.abs().max()


@pytest.mark.parametrize("cache_dtype", ["int8", "float8_e4m3fn"])
def test_generation_and_memory(cache_dtype):
    lm, config = model("tiny", "d", cache_dtype)
    whole, _ = model("tiny", "d", None)
    prompts = [[5, 17, 3], [9], list(range(100))]
    out = lm.generate_batch(prompts, 20, eos=[])
    assert [len(o) for o in out] == [20, 20, 20] and out == lm.generate_batch(prompts, 20, eos=[])
    assert lm.generate(prompts[2], 20) == lm.generate(prompts[2], 20)
    size = lambda m: sum(t.numel() * t.element_size() for g in m.engine.cache.groups for t in (g.keys, g.values, g.key_scales, g.value_scales) if t is not None)
    assert size(lm) * 128 == size(whole) * 68                        # 64 codes and a scale for 64 entries of two bytes


def test_command_line_and_replay(tmp_path):
    from tiny_configs import CONFIG_B, INIT_B
    folder = str(tmp_path / "model")
    fr.write_random_model(folder, CONFIG_B, INIT_B)
    ids = tmp_path / "ids.json"
    ids.write_text(json.dumps({"holdout_ids": list(range(30))}))
    run = lambda *args, **more: subprocess.run([sys.executable, *args], cwd=ROOT, capture_output=True, text=True, timeout=600, **more)
    want = fr.load(folder, max_tokens=64, cache_dtype="int8").generate(list(range(12)), 6)
    proc = run("-m", "fieldrun_b200", "--model", folder, "--ids", str(ids), "--ctx", "12", "--generate", "6", "--eos", "none", "--cache-dtype", "int8")
    assert proc.returncode == 0, proc.stderr[-2000:]
    assert " ".join(map(str, want)) in proc.stdout
    proc = run("-m", "fieldrun_b200", "--model", folder, "--ids", str(ids), "--ctx", "12", "--generate", "6", "--dtype", "float32", "--cache-dtype", "int8")
    assert proc.returncode == 1 and "for bfloat16 models" in proc.stderr
    out = str(tmp_path / "out")
    step = {"step": 0, "entries": [{"id": "a", "tokens": list(range(12)), "want": [11]}], "end": []}
    proc = run(os.path.join(ROOT, "bin", "trace_run"), "--model", folder, "--dtype", "bfloat16", "--out", out, "--max-tokens", "64", "--cache-dtype", "int8",
               input=json.dumps(step) + "\n")
    assert proc.returncode == 0, proc.stderr[-2000:]
    logits = np.fromfile(os.path.join(out, "0.f32"), dtype="<f4")
    assert int(logits.argmax()) == want[0]


@pytest.mark.parametrize("design,name", MODELS)
def test_pages_read_back_in_portions_give_the_same_bits(design, name, monkeypatch):
    # steps that mix prompts with single tokens over longer histories, the read-back in one portion and in several
    from fieldrun_b200.parts import attention
    logits, rooms = [], []
    for most in (attention.READ_BACK_BYTES, 1 << 17):
        monkeypatch.setattr(attention, "READ_BACK_BYTES", most)
        lm, config = model(design, name, "int8")
        engine = lm.engine
        rng = np.random.default_rng(11)
        draw = lambda n: rng.integers(0, vocabulary(config), size=n).tolist()
        slots = [engine.new_sequence() for _ in range(6)]
        out = [engine.step(slots, [draw(n) for n in (400, 9, 200, 1, 130, 333)])]
        out.append(engine.step(slots, [draw(n) for n in (1, 1, 70, 1, 1, 1)]))
        out.append(engine.step(slots, [draw(n) for n in (1, 1, 1, 5, 1, 1)]))
        engine.check()
        logits.append(torch.cat(out).cpu())
        rooms.append(sum(engine.workspace.buffer(n, (0,), torch.bfloat16).untyped_storage().nbytes() for n in ("attention.keys", "attention.values")))
    assert torch.isfinite(logits[0]).all() and torch.equal(*logits)
    assert rooms[1] < rooms[0]
