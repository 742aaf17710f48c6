"""Products in 8-bit integers, as cases that can be timed and compared: a linear layer, a gated feed-forward block, routed experts.

A weight's row (an output channel) and a token's row are held as 8-bit integers with one float32 scale each,

    scale = max |x| / 127,  code = x * 127 / max |x| rounded half to even,

and a product is  out[t, f] = scale_x[t] * scale_w[f] * sum_k code_x[t, k] code_w[f, k]  with a sum of whole numbers.

linear:   out = x W^T, x rounded to codes token by token.
gated:    h = act(x W_gate^T) * (x W_up^T) in 32 bits, rounded to codes token by token;  out = h W_down^T.
          act: silu or gelu_tanh; with a limit L the clamped gate  g = min(gate, L), u = clamp(up, -L, L), g sigmoid(1.702 g) (u + 1).
experts:  every token goes through the gated blocks of its experts; out = sum over its experts of weight * block(x).

Weights lie as codes [experts, 1 or 2 (gate, up), rows, entries] with rows and entries filled up with zeros to multiples of 16 and 128, and
scales [experts, 1 or 2, rows].  ``run`` computes in elementary torch operations while ``own`` is false and calls the framework's operators
while it is true.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPE = {"bfloat16": torch.bfloat16, "float32": torch.float32}
SLOPE = 1.702


def _case(name, op, rows, inner, width, x="bfloat16", out="float32", **more):
    """linear: ``inner`` entries in, ``width`` out; gated and experts: ``inner`` entries in and out, ``width`` between."""
    case = dict(op=op, rows=rows, inner=inner, width=width, x=x, out=out, activation="silu", limit=0.0, experts=1, top_k=1)
    case.update(more)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # the smallest call: one conversation's next token through a small layer's output projection
        _case("linear_1_token_1024", "linear", 1, 1024, 1024),
        # one token through the query, key and value projections of a larger layer
        _case("linear_1_token_4096", "linear", 1, 4096, 6144),
        # a serving batch's next tokens
        _case("linear_24_tokens", "linear", 24, 4096, 14336),
        # odd sizes everywhere, rows in 32 bits (a normed stream), results in 16
        _case("linear_ragged", "linear", 77, 1000, 1999, x="float32", out="bfloat16"),
        # a prompt through a square projection
        _case("linear_prompt_2048", "linear", 2048, 4096, 4096),
        # several prompts in one step through a wide projection
        _case("linear_prompts_8192", "linear", 8192, 4096, 12288, out="bfloat16"),
        # one token's feed-forward
        _case("gated_1_token", "gated", 1, 4096, 12288, out="bfloat16"),
        # odd sizes and the other activation
        _case("gated_ragged_gelu", "gated", 301, 2000, 5502, x="float32", out="bfloat16", activation="gelu_tanh"),
        # a prompt's feed-forward
        _case("gated_prompt_2048", "gated", 2048, 4096, 8192, out="bfloat16"),
        # eight conversations' next tokens through MiniMax-M2's experts
        _case("experts_8_tokens_m2", "experts", 8, 3072, 1536, out="bfloat16", experts=256, top_k=8),
        # odd sizes and the clamped gate
        _case("experts_ragged_clamped", "experts", 130, 1000, 504, out="bfloat16", experts=20, top_k=3, limit=7.0),
        # a prompt through the experts of a smaller layer
        _case("experts_prompt_2048", "experts", 2048, 2048, 1024, out="bfloat16", experts=64, top_k=8),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    def size(low, high):                       # a model's sizes are mostly round, and sometimes not
        n = spread(low, high)
        return max(low, n // 128 * 128) if rng.random() < 0.6 else n
    op = rng.choice(["linear", "linear", "gated", "experts"])
    x = rng.choice(["bfloat16", "bfloat16", "float32"])
    while True:
        if op == "linear":
            case = _case(None, op, spread(1, 8192), size(256, 8192), size(256, 16384), x, rng.choice(["float32", "bfloat16"]))
        elif op == "gated":
            case = _case(None, op, spread(1, 2048), size(256, 4096), size(256, 12288), x, "bfloat16",
                         activation=rng.choice(["silu", "silu", "gelu_tanh"]))
            if rng.random() < 0.2:
                case.update(activation="silu", limit=rng.choice([5.0, 7.0]))
        else:
            experts = spread(4, 256)
            case = _case(None, op, spread(1, 2048), size(256, 2048), size(128, 1536), x, "bfloat16", experts=experts,
                         top_k=rng.randint(1, min(8, experts)), limit=rng.choice([0.0, 0.0, 7.0]))
        need = work(case)
        if need["flops"] <= 4.2e11 and need["bytes"] <= 1.2e9:
            return case


# ------------------------------------------------------------------------------------------------ inputs

def _up(n, step):
    return -(-n // step) * step


def _weight(gen, experts, parts, rows, inner):
    """A trained layer's weights, about N(0, 1 / inner) with rows of unlike size, as codes and scales in their layout."""
    codes = torch.zeros((experts, parts, _up(rows, 16), _up(inner, 128)), dtype=torch.int8, device=DEVICE)
    scales = torch.zeros((experts, parts, _up(rows, 16)), dtype=torch.float32, device=DEVICE)
    per_go = max(1, (1 << 28) // (parts * rows * inner))
    for e in range(0, experts, per_go):
        n = min(per_go, experts - e)
        w = torch.randn((n, parts, rows, inner), generator=gen, device=DEVICE)
        w *= torch.exp(0.3 * torch.randn((n, parts, rows, 1), generator=gen, device=DEVICE)) / math.sqrt(inner)
        top = w.abs().amax(-1, keepdim=True)
        codes[e:e + n, :, :rows, :inner] = torch.round(w * (127.0 / top)).to(torch.int8)
        scales[e:e + n, :, :rows] = (top / 127.0).squeeze(-1)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    rows, inner, width = case["rows"], case["inner"], case["width"]
    # normed rows: about one in size, some channels several times as large as the others
    gain = torch.exp(0.4 * torch.randn(inner, generator=gen, device=DEVICE))
    gain[torch.randperm(inner, generator=gen, device=DEVICE)[:max(1, inner // 200)]] *= 8.0
    x = (torch.randn((rows, inner), generator=gen, device=DEVICE) * gain).to(TYPE[case["x"]])
    s = dict(case=case, x=x)
    if case["op"] == "linear":
        s["w"], s["w_scale"] = _weight(gen, 1, 1, width, inner)
        return s
    s["w_in"], s["w_in_scale"] = _weight(gen, case["experts"], 2, width, inner)
    s["w_down"], s["w_down_scale"] = _weight(gen, case["experts"], 1, inner, width)
    if case["op"] == "experts":                # a router's choice: some experts are picked several times as often as others
        liking = torch.randn((rows, case["experts"]), generator=gen, device=DEVICE) \
            + 0.7 * torch.randn(case["experts"], generator=gen, device=DEVICE)
        top, ids = liking.topk(case["top_k"], dim=-1)
        s["ids"], s["weights"] = ids.to(torch.int32), torch.softmax(top, -1)
    return s


# ------------------------------------------------------------------------------------------------ the plain form

def _plain_codes(x):
    """Codes (as numbers) and scale of every row; in 64 bits, where a value next to a border goes to its side."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    safe = torch.where(top > 0, top, 1.0)
    return torch.round(x * 127.0 / safe).float(), (top / 127.0).float()


def _plain_product(x, codes, scales):
    """x [.., T, K] with codes [.., F, K] and scales [.., F]."""
    q, scale = _plain_codes(x)
    return (q @ codes.float().transpose(-1, -2)) * scale * scales.unsqueeze(-2)


def _plain_gate(gate, up, activation, limit):
    if limit > 0.0:
        g, u = gate.clamp(max=limit), up.clamp(-limit, limit)
        return g / (1.0 + torch.exp(-SLOPE * g)) * (u + 1.0)
    if activation == "gelu_tanh":
        return 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate * gate * gate))) * up
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain_block(case, x, w_in, w_in_scale, w_down, w_down_scale):
    """The gated block of one expert, or of each of several side by side (a leading dimension everywhere)."""
    inner, width = case["inner"], case["width"]
    gate = _plain_product(x, w_in[..., 0, :width, :inner], w_in_scale[..., 0, :width])
    up = _plain_product(x, w_in[..., 1, :width, :inner], w_in_scale[..., 1, :width])
    hidden = _plain_gate(gate, up, case["activation"], case["limit"])
    return _plain_product(hidden, w_down[..., 0, :inner, :width], w_down_scale[..., 0, :inner])


def _plain_experts(case, s):
    x, ids, (rows, top_k) = s["x"], s["ids"].long(), s["ids"].shape
    flat = ids.reshape(-1)
    if flat.numel() <= case["experts"]:        # few tokens: every token's experts by themselves
        y = _plain_block(case, x.repeat_interleave(top_k, 0).unsqueeze(1), s["w_in"][flat], s["w_in_scale"][flat], s["w_down"][flat], s["w_down_scale"][flat])
        y = y.squeeze(1)
    else:                                      # every expert's tokens side by side, filled up to the most that one has
        order = flat.argsort(stable=True)
        counts = torch.bincount(flat, minlength=case["experts"])
        place = torch.arange(flat.numel(), device=DEVICE) - (counts.cumsum(0) - counts)[flat[order]]
        side = torch.zeros((case["experts"], int(counts.max()), case["inner"]), dtype=x.dtype, device=DEVICE)
        side[flat[order], place] = x[order // top_k]
        done = _plain_block(case, side, s["w_in"], s["w_in_scale"], s["w_down"], s["w_down_scale"])
        y = torch.empty((flat.numel(), case["inner"]), device=DEVICE)
        y[order] = done[flat[order], place]
    return (y.view(rows, top_k, -1) * s["weights"].unsqueeze(-1)).sum(1)


def _plain(s):
    case = s["case"]
    if case["op"] == "linear":
        out = _plain_product(s["x"], s["w"][0, 0, :case["width"], :case["inner"]], s["w_scale"][0, 0, :case["width"]])
    elif case["op"] == "gated":
        out = _plain_block(case, s["x"], s["w_in"][0], s["w_in_scale"][0], s["w_down"][0], s["w_down_scale"][0])
    else:
        out = _plain_experts(case, s)
    return out.to(TYPE[case["out"]])


# ------------------------------------------------------------------------------------------------ the framework's operators

def _own(s):
    from fieldrun_b200.csrc import ops
    case, x = s["case"], s["x"]
    features = case["width"] if case["op"] == "linear" else case["inner"]
    out = torch.empty((case["rows"], features), dtype=TYPE[case["out"]], device=DEVICE)
    if case["op"] == "linear":
        ops.linear_8bit(x, s["w"], s["w_scale"], out)
    elif case["op"] == "gated":
        ops.gated_8bit(x, s["w_in"], s["w_in_scale"], s["w_down"], s["w_down_scale"], out, width=case["width"], activation=case["activation"],
                       gate_limit=case["limit"])
    else:
        ops.experts_8bit(x, s["ids"], s["weights"], s["w_in"], s["w_in_scale"], s["w_down"], s["w_down_scale"], out, width=case["width"],
                         gate_limit=case["limit"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    rows, inner, width, experts, top_k = (case[n] for n in ("rows", "inner", "width", "experts", "top_k"))
    size = {"bfloat16": 2, "float32": 4}
    if case["op"] == "linear":
        return {"bytes": rows * (inner * size[case["x"]] + width * size[case["out"]]) + width * (inner + 4), "flops": 2 * rows * inner * width}
    touched = experts * (1.0 - (1.0 - top_k / experts) ** rows) if case["op"] == "experts" else 1
    weights = touched * (3 * inner * width + 4 * (2 * width + inner))
    routing = rows * top_k * 8 if case["op"] == "experts" else 0
    return {"bytes": int(rows * inner * (size[case["x"]] + size[case["out"]]) + weights + routing), "flops": 6 * rows * top_k * inner * width}


# ------------------------------------------------------------------------------------------------ in 64 bits

def _rounded(x):
    largest = torch.amax(torch.abs(x), dim=1, keepdim=True)
    step = largest / 127
    codes = torch.where(largest > 0, torch.round(127 * x / torch.clamp(largest, min=1e-300)), torch.zeros_like(x))
    return codes, step


def _exact_linear(x, codes, scales, rows, inner):
    q, step = _rounded(x)
    return torch.mm(q, codes[:rows, :inner].double().t()) * step * scales[:rows].double()


def _exact_unit(case, x, w_in, in_scale, w_down, down_scale):
    inner, width, limit = case["inner"], case["width"], case["limit"]
    a = _exact_linear(x, w_in[0], in_scale[0], width, inner)
    b = _exact_linear(x, w_in[1], in_scale[1], width, inner)
    if limit > 0:
        a = torch.minimum(a, torch.full_like(a, limit))
        h = a * torch.sigmoid(SLOPE * a) * (torch.clamp(b, min=-limit, max=limit) + 1)
    elif case["activation"] == "gelu_tanh":
        h = a * b / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (a + 0.044715 * a ** 3)))
    else:
        h = a * torch.sigmoid(a) * b
    return _exact_linear(h, w_down[0], down_scale[0], inner, width)


def exact(case, seed):
    if work(case)["flops"] > 2e13:             # at least a second of products in 64 bits
        return None
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "linear":
        return _exact_linear(x, s["w"][0, 0], s["w_scale"][0, 0], case["width"], case["inner"])
    if case["op"] == "gated":
        return _exact_unit(case, x, s["w_in"][0], s["w_in_scale"][0], s["w_down"][0], s["w_down_scale"][0])
    out = torch.zeros((case["rows"], case["inner"]), dtype=torch.float64, device=DEVICE)
    for e in range(case["experts"]):
        token, rank = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel():
            unit = _exact_unit(case, x[token], s["w_in"][e], s["w_in_scale"][e], s["w_down"][e], s["w_down_scale"][e])
            out.index_add_(0, token, unit * s["weights"][token, rank].double().unsqueeze(1))
    return out
