"""A key-value cache held in 8 bits, as cases that can be timed and compared: projections written into it, its pages read
back, one token's attention over it.

A row (one token's key or value of one head) is stored as 8-bit codes with one float32 scale: scale = max |x| / Q and
code = x * Q / max |x| rounded to the type, half to even, with Q = 448 for float8_e4m3fn and 127 for int8.  Pages hold 64
tokens: codes [pages, heads, 64, entries], scales [pages, heads, 64]; a table names the page of (sequence, position // 64).

``run`` computes the operators in elementary torch operations while ``own`` is false and calls the framework's while it is true.
"""
import math

import torch

own = False

DEVICE = "cuda"
PAGE = 64
CHUNK = 256                       # keys that a partial result of the one-token attention covers at least
EPS = 1e-6
LIMIT = {"float8_e4m3fn": 448.0, "int8": 127.0}
TYPE = {"float8_e4m3fn": torch.float8_e4m3fn, "int8": torch.int8}
SMALLEST = 2.0 ** -96             # a row whose largest entry is below this is stored as zeros

# query heads, key heads, key size, value size, maps per head: MiniMax-M2's layer, the smaller layers of the other designs,
# differential attention (two maps share a value head; query and key heads counted with their maps)
HEADS = {"m2": (48, 8, 128, 128, 1), "w2048": (16, 4, 128, 128, 1), "w1024": (16, 4, 64, 64, 1), "narrow": (12, 4, 32, 32, 1),
         "odd": (12, 2, 96, 96, 1), "pair": (32, 8, 64, 128, 2), "shared": (24, 1, 128, 128, 1)}


def _case(name, op, heads, storage, seqs, longest, shortest=None, **more):
    case = dict(op=op, heads=heads, storage=storage, seqs=seqs, longest=longest, shortest=longest if shortest is None else shortest,
                norm="none", rotary=0, interleaved=False, window=0, chunk=0, keep_first=0, sinks=False, slopes=False, softcap=0.0)
    case.update(more)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # the smallest call: one conversation's next token through MiniMax-M2's projections into the cache
        _case("write_one_token", "write", "m2", "float8_e4m3fn", 1, 1, norm="full_width", rotary=64),
        # 64 conversations' next tokens
        _case("write_64_tokens", "write", "m2", "float8_e4m3fn", 64, 1, norm="full_width", rotary=64),
        # a prompt of 2,048 tokens written, and read back for the prompt's attention
        _case("prompt_2048_int8", "prompt", "m2", "int8", 1, 2048, norm="full_width", rotary=64),
        # a ragged batch of prompts through a smaller layer with a norm per head and paired rotation
        _case("prompts_ragged", "prompt", "w1024", "float8_e4m3fn", 9, 3001, 1, norm="per_head", rotary=64, interleaved=True),
        # a long history read back, for a prompt that goes on behind it
        _case("read_32768", "read", "m2", "float8_e4m3fn", 1, 32768),
        # the last windows of a ragged batch read back
        _case("read_windows_int8", "read", "w2048", "int8", 16, 20011, 77, window=4096),
        # one token over a short and over a very long conversation: latency, and the split over the length
        _case("token_1x2048", "token", "m2", "float8_e4m3fn", 1, 2048),
        _case("token_1x131072_int8", "token", "m2", "int8", 1, 131072),
        # a serving batch over caches of one length
        _case("token_32x4096", "token", "m2", "float8_e4m3fn", 32, 4096),
        # a ragged batch with everything that changes a score: window with first tokens, sinks, capped scores
        _case("token_64_ragged_int8", "token", "w1024", "int8", 64, 16384, 1, window=8000, keep_first=4, sinks=True, softcap=30.0),
        # differential attention: two maps a head over shared values
        _case("token_16_pair", "token", "pair", "float8_e4m3fn", 16, 12345, 500),
        # a whole decode step of the cache: eight conversations' tokens written, then attended over
        _case("step_8_ragged", "step", "m2", "float8_e4m3fn", 8, 32768, 3000, norm="full_width", rotary=64),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["write", "prompt", "read", "token", "token", "step"])
    heads = rng.choice(sorted(HEADS))
    size = HEADS[heads][2]
    storage = rng.choice(sorted(LIMIT)) if op in ("prompt", "read", "token") else "float8_e4m3fn"
    norm = rng.choice(["none", "per_head", "full_width"]) if heads != "pair" else "none"
    rotary = rng.choice([0, size // 2, size])
    interleaved = rng.random() < 0.5
    if op == "write":
        return _case(None, op, heads, storage, spread(1, 256), 1, norm=norm, rotary=rotary, interleaved=interleaved)
    if op == "prompt":
        seqs = spread(1, 16)
        longest = spread(3, 12000 // seqs)
        return _case(None, op, heads, storage, seqs, longest, rng.randint(1, longest), norm=norm, rotary=rotary, interleaved=interleaved)
    window = rng.choice([0, 0, spread(50, 10000)])
    chunk = spread(50, 10000) if not window and rng.random() < 0.3 else 0
    keep_first = rng.randint(1, 200) if window and rng.random() < 0.5 else 0
    seqs = spread(1, 64)
    # lengths whose keys and values stay below the largest listed case's
    entries = HEADS[heads][1] * size * seqs
    longest = spread(20, max(21, min(131072, 100_000_000 // entries)))
    extras = dict(window=window, chunk=chunk, keep_first=keep_first)
    if op == "read":
        return _case(None, op, heads, storage, seqs, longest, rng.randint(1, longest), **extras)
    if heads != "pair":
        extras.update(sinks=rng.random() < 0.3, slopes=rng.random() < 0.3)
    extras.update(softcap=rng.choice([0.0, 0.0, 30.0]))
    if op == "step":
        extras.update(norm=norm, rotary=rotary, interleaved=interleaved)
    return _case(None, op, heads, storage, seqs, longest, rng.randint(1, longest), **extras)


# ------------------------------------------------------------------------------------------------ sizes of a case

def _sizes(case):
    q_heads, k_heads, dim, vdim, maps = HEADS[case["heads"]]
    return q_heads, k_heads, k_heads // maps, dim, vdim, maps


def _lengths(case):
    """Tokens that each sequence holds once the case has run, from the longest down, the middle ones closer to the shortest."""
    n, hi, lo = case["seqs"], case["longest"], case["shortest"]
    return [lo + (hi - lo) * (n - 1 - i) ** 2 // max(1, (n - 1) ** 2) if n > 1 else hi for i in range(n)]


def _starts(case):
    """Positions of each sequence's first new token: prompts begin at 0, single tokens are the last ones held."""
    if case["op"] == "prompt":
        return [0] * case["seqs"]
    if case["op"] == "write":                          # tokens at unequal places of long conversations
        return [(977 * i + 301) % 4096 for i in range(case["seqs"])]
    return [n - 1 for n in _lengths(case)]


def _first_key(case, position):
    lo = max(0, position - case["window"] + 1) if case["window"] else 0
    return max(lo, position // case["chunk"] * case["chunk"]) if case["chunk"] else lo


def _pages_in_sight(case):
    """(sequence, page number) of every page that the tokens from each sequence's first new one on may see."""
    found = []
    for seq, (start, length) in enumerate(zip(_starts(case), _lengths(case))):
        first = _first_key(case, start) // PAGE
        kept = min(-(-case["keep_first"] // PAGE), first)
        found += [(seq, p) for p in range(kept)] + [(seq, p) for p in range(first, (length - 1) // PAGE + 1)]
    return found


def _visible(case):
    """Keys that the case's single tokens see, summed over the sequences."""
    total = 0
    for start in _starts(case):
        first = _first_key(case, start)
        total += start + 1 - first + min(case["keep_first"], first)
    return total


def work(case):
    q_heads, k_heads, v_heads, dim, vdim, maps = _sizes(case)
    op, lengths = case["op"], _lengths(case)
    tokens = sum(lengths) if op == "prompt" else case["seqs"]
    row = (q_heads + k_heads) * dim + v_heads * vdim
    stored = k_heads * (dim + 4) + v_heads * (vdim + 4)                       # bytes that a token takes in the cache
    moved = flops = 0
    if op in ("write", "prompt", "step"):
        moved += tokens * (4 * row + 2 * q_heads * dim + stored + 4 * case["rotary"])
        flops += tokens * row * 8
    if op == "prompt":
        moved += len(_pages_in_sight(case)) * PAGE * 2 * (k_heads * dim + v_heads * vdim)
    if op == "read":
        moved += len(_pages_in_sight(case)) * PAGE * (stored + 2 * (k_heads * dim + v_heads * vdim))
        flops += len(_pages_in_sight(case)) * PAGE * (k_heads * dim + v_heads * vdim)
    if op in ("token", "step"):
        moved += _visible(case) * stored + tokens * 2 * (q_heads * dim + q_heads // maps * vdim)
        flops += _visible(case) * q_heads * 2 * (dim + vdim)
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------------------------ inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _store(x, storage):
    """The codes and scales of rows x [..., entries] in float32."""
    top = x.abs().amax(-1, keepdim=True)
    empty = top < SMALLEST
    scaled = x * torch.where(empty, torch.zeros_like(top), LIMIT[storage] / top)
    codes = scaled.to(torch.float8_e4m3fn) if storage == "float8_e4m3fn" else scaled.round().to(torch.int8)
    return codes, torch.where(empty, torch.zeros_like(top), top / LIMIT[storage]).squeeze(-1)


def _drawn_pages(gen, pages, heads, size, storage, spread):
    """A page store as a conversation leaves it: rows whose sizes differ by ``spread`` (keys have a few entries far above the
    others), put into codes by pieces so that the float32 rows never lie there all at once."""
    codes = torch.empty((pages, heads, PAGE, size), dtype=TYPE[storage], device=DEVICE)
    scales = torch.empty((pages, heads, PAGE), dtype=torch.float32, device=DEVICE)
    channel = torch.exp(spread * torch.randn(heads, 1, size, device=DEVICE, generator=gen))
    for at in range(0, pages, 2048):
        part = codes[at:at + 2048]
        x = torch.randn(part.shape, device=DEVICE, generator=gen) * channel
        x *= torch.exp(0.3 * torch.randn((*part.shape[:3], 1), device=DEVICE, generator=gen))
        codes[at:at + 2048], scales[at:at + 2048] = _store(x, storage)
    return codes, scales


def prepare(case, seed):
    q_heads, k_heads, v_heads, dim, vdim, maps = _sizes(case)
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(1_000_003 * (seed + 1))
    storage, op, seqs = case["storage"], case["op"], case["seqs"]
    lengths, starts = _lengths(case), _starts(case)
    held = [start + 1 for start in starts] if op == "write" else lengths
    new = lengths if op == "prompt" else [1] * seqs
    counts = [-(-n // PAGE) for n in held]
    # a page for every number in use, in no order; slots in another order than the sequences
    if op == "write":
        pages, order = seqs, torch.randperm(seqs, device=DEVICE, generator=gen)
    else:
        pages = sum(counts)
        order = torch.randperm(pages, device=DEVICE, generator=gen)
    slots = torch.randperm(seqs, device=DEVICE, generator=gen)
    table = torch.full((seqs, max(counts)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, count in enumerate(counts):
        if op == "write":
            table[slots[i], count - 1] = order[i]
        else:
            table[slots[i], :count] = order[at:at + count]
            at += count
    s = dict(case=case, table=table, slot=slots.to(torch.int32), start=_ints(starts), new=_ints(new),
             tok_pos=torch.cat([torch.arange(a, a + n, device=DEVICE) for a, n in zip(starts, new)]).to(torch.int32),
             tok_slot=torch.repeat_interleave(slots, torch.tensor(new, device=DEVICE)).to(torch.int32))
    tokens = sum(new)
    if op in ("read", "token", "step"):
        s["k"], s["k_scale"] = _drawn_pages(gen, pages, k_heads, dim, storage, 0.7)
        s["v"], s["v_scale"] = _drawn_pages(gen, pages, v_heads, vdim, storage, 0.2)
    else:
        s["k"] = torch.zeros((pages, k_heads, PAGE, dim), device=DEVICE).to(TYPE[storage])
        s["v"] = torch.zeros((pages, v_heads, PAGE, vdim), device=DEVICE).to(TYPE[storage])
        s["k_scale"] = torch.zeros((pages, k_heads, PAGE), device=DEVICE)
        s["v_scale"] = torch.zeros((pages, v_heads, PAGE), device=DEVICE)
    if op in ("write", "prompt", "step"):
        row = (q_heads + k_heads) * dim + v_heads * vdim
        s["qkv"] = torch.randn(tokens, row, device=DEVICE, generator=gen) * torch.exp(0.5 * torch.randn(row, device=DEVICE, generator=gen))
        width = dict(none=(0, 0), per_head=(dim, dim), full_width=(q_heads * dim, k_heads * dim))[case["norm"]]
        s["q_norm"], s["k_norm"] = (1 + 0.1 * torch.randn(w, device=DEVICE, generator=gen) if w else None for w in width)
        if case["rotary"]:
            half = case["rotary"] // 2
            angle = torch.arange(max(held), dtype=torch.float64, device=DEVICE)[:, None] * 1e6 ** (
                -torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
            s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        else:
            s["cos"] = s["sin"] = None
        s["q_out"] = torch.empty((tokens, q_heads * dim), dtype=torch.bfloat16, device=DEVICE)
    if op in ("prompt", "read"):
        sight = _pages_in_sight(case)
        s["page_seq"], s["page_index"] = _ints([a for a, _ in sight]), _ints([b for _, b in sight])
        s["keys"] = torch.empty((len(sight), k_heads, PAGE, dim), dtype=torch.bfloat16, device=DEVICE)
        s["values"] = torch.empty((len(sight), v_heads, vdim, PAGE), dtype=torch.bfloat16, device=DEVICE)
    if op in ("token", "step"):
        if op == "token":
            s["q"] = torch.randn(seqs, q_heads * dim, device=DEVICE, generator=gen).to(torch.bfloat16)
        s["sinks"] = torch.randn(q_heads, device=DEVICE, generator=gen) if case["sinks"] else None
        s["slopes"] = 2.0 ** torch.linspace(-2.0, -12.0, q_heads, device=DEVICE) if case["slopes"] else None
        s["lam"] = torch.full((1,), 0.3, device=DEVICE) + 0.1 * torch.rand(1, device=DEVICE, generator=gen) if maps == 2 else None
        chunks = -(-max(lengths) // CHUNK)
        s["part_o"] = torch.empty((seqs, q_heads, chunks, vdim), dtype=torch.float32, device=DEVICE)
        s["part_ml"] = torch.empty((seqs, q_heads, chunks, 2), dtype=torch.float32, device=DEVICE)
        s["out"] = torch.empty((seqs, q_heads // maps * vdim), dtype=torch.bfloat16, device=DEVICE)
        s["max_chunks"] = chunks
    return s


# ------------------------------------------------------------------------------------------------ plain forms

DIFF_EPS, DIFF_FACTOR = 1e-6, 0.8


def _rotate(x, s):
    """x [T, heads, size] with its first rotary entries turned by the angles of the tokens' positions."""
    rot = s["case"]["rotary"]
    if not rot:
        return x
    cos, sin = s["cos"][s["tok_pos"].long()][:, None], s["sin"][s["tok_pos"].long()][:, None]
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if s["case"]["interleaved"] else (r[..., :rot // 2], r[..., rot // 2:])
    turned = (a * cos - b * sin, b * cos + a * sin)
    r = torch.stack(turned, -1).flatten(-2) if s["case"]["interleaved"] else torch.cat(turned, -1)
    return torch.cat([r, x[..., rot:]], -1)


def _plain_write(s):
    q_heads, k_heads, v_heads, dim, vdim, _ = _sizes(s["case"])
    tokens = s["qkv"].shape[0]
    q, k, v = s["qkv"].split([q_heads * dim, k_heads * dim, v_heads * vdim], -1)
    if s["case"]["norm"] == "full_width":
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    q, k, v = q.reshape(tokens, q_heads, dim), k.reshape(tokens, k_heads, dim), v.reshape(tokens, v_heads, vdim)
    if s["case"]["norm"] == "per_head":
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    s["q_out"].copy_(_rotate(q, s).reshape(tokens, -1))
    position = s["tok_pos"].long()
    page, place = s["table"][s["tok_slot"].long(), position // PAGE].long(), position % PAGE
    for_k, for_v = _store(_rotate(k, s), s["case"]["storage"]), _store(v, s["case"]["storage"])
    _bytes(s["k"]).transpose(1, 2)[page, place], s["k_scale"].transpose(1, 2)[page, place] = _bytes(for_k[0]), for_k[1]
    _bytes(s["v"]).transpose(1, 2)[page, place], s["v_scale"].transpose(1, 2)[page, place] = _bytes(for_v[0]), for_v[1]


def _bytes(codes):
    """Codes as bytes: what moves them about has no form for 8-bit floating types everywhere."""
    return codes.view(torch.uint8)


def _values(s, name, page):
    """The rows of whole pages in float32."""
    return _bytes(s[name])[page].view(s[name].dtype).float() * s[name + "_scale"][page][..., None]


def _plain_read(s):
    seq = s["page_seq"].long()
    page = s["table"][s["slot"][seq].long(), s["page_index"].long()].long()
    token = s["page_index"][:, None] * PAGE + torch.arange(PAGE, device=DEVICE)
    there = (token < (s["start"] + s["new"])[seq][:, None])[:, None, :, None]
    keys = _values(s, "k", page)
    values = _values(s, "v", page)
    s["keys"].copy_(torch.where(there, keys, torch.zeros_like(keys)))
    s["values"].copy_(torch.where(there, values, torch.zeros_like(values)).transpose(2, 3))


def _plain_attend(s, q):
    case = s["case"]
    q_heads, k_heads, v_heads, dim, vdim, maps = _sizes(case)
    seqs, longest, group = case["seqs"], max(_lengths(case)), q_heads // k_heads
    held = -(-longest // PAGE)
    page = s["table"][s["slot"].long(), :held].long().clamp_min(0)                     # [sequence, page number]
    k = _values(s, "k", page).transpose(1, 2).reshape(seqs, k_heads, held * PAGE, dim)
    position, key = s["start"][:, None].long(), torch.arange(held * PAGE, device=DEVICE)[None]
    score = torch.matmul(q.float().reshape(seqs, k_heads, group, dim), k.transpose(2, 3)) * dim ** -0.5
    del k
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    if s["slopes"] is not None:
        score = score + s["slopes"].reshape(k_heads, group)[None, :, :, None] * (key - position)[:, None, None, :]
    lo = torch.zeros_like(position)
    if case["window"]:
        lo = (position - case["window"] + 1).clamp_min(0)
    if case["chunk"]:
        lo = torch.maximum(lo, position // case["chunk"] * case["chunk"])
    seen = (key <= position) & ((key >= lo) | (key < case["keep_first"]))
    score = torch.where(seen[:, None, None, :], score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].reshape(1, k_heads, group, 1)
        top = torch.maximum(top, sink)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    del score
    v = _values(s, "v", page).transpose(1, 2).reshape(seqs, v_heads, held * PAGE, vdim)
    v = torch.where(seen[:, None, :, None], v, torch.zeros_like(v))
    out = torch.matmul(weight.reshape(seqs, v_heads, maps * group, held * PAGE), v).reshape(seqs, v_heads, maps, group, vdim)
    out = out / total.reshape(seqs, v_heads, maps, group, 1)
    if maps == 2:
        out = out[:, :, 0] - s["lam"] * out[:, :, 1]
        out = out * torch.rsqrt(out.square().mean(-1, keepdim=True) + DIFF_EPS) * DIFF_FACTOR
    s["out"].copy_(out.reshape(seqs, -1))


# ------------------------------------------------------------------------------------------------ one pass

def _own_write(s):
    from fieldrun_b200.csrc import ops
    q_heads, k_heads, v_heads, dim, vdim, _ = _sizes(s["case"])
    ops.qkv_prepare_8bit(s["qkv"], s["q_norm"], s["k_norm"], EPS, s["cos"], s["sin"], s["tok_pos"], s["tok_slot"], s["table"],
                         s["q_out"], s["k"], s["k_scale"], s["v"], s["v_scale"], num_heads=q_heads, num_kv_heads=k_heads,
                         num_v_heads=v_heads, head_dim=dim, v_dim=vdim, rotary_dim=s["case"]["rotary"],
                         interleaved=s["case"]["interleaved"], per_head=s["case"]["norm"] == "per_head")


def _own_read(s):
    from fieldrun_b200.csrc import ops
    ops.cache_read_8bit(s["k"], s["k_scale"], s["v"], s["v_scale"], s["table"], s["page_seq"], s["page_index"], s["slot"], s["start"],
                        s["new"], s["keys"], s["values"])


def _own_attend(s, q):
    from fieldrun_b200.csrc import ops
    case = s["case"]
    q_heads, k_heads, v_heads, dim, vdim, maps = _sizes(case)
    ops.attention_decode_8bit(q, s["k"], s["k_scale"], s["v"], s["v_scale"], s["table"], s["start"], s["slot"], s["part_o"], s["part_ml"],
                              s["out"], num_heads=q_heads, num_kv_heads=k_heads, head_dim=dim, v_dim=vdim, scale=dim ** -0.5,
                              window=case["window"] or None, chunk=case["chunk"] or None, keep_first=case["keep_first"],
                              max_chunks=s["max_chunks"], slopes=s["slopes"], sinks=s["sinks"], softcap=case["softcap"] or None, maps=maps,
                              pages_final=True,               # at most one row a sequence was just written, into its newest page
                              difference=dict(lam=s["lam"], eps=DIFF_EPS, factor=DIFF_FACTOR) if maps == 2 else None)


def run(s):
    op = s["case"]["op"]
    write, read, attend = (_own_write, _own_read, _own_attend) if own else (_plain_write, _plain_read, _plain_attend)
    out = {}
    if op in ("write", "prompt", "step"):
        write(s)
        out.update(q=s["q_out"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        if op != "prompt":
            out.update(k=s["k"], v=s["v"])
    if op in ("prompt", "read"):
        read(s)
        out.update(keys=s["keys"], values=s["values"])
    if op in ("token", "step"):
        attend(s, s["q"] if op == "token" else s["q_out"])
        out.update(out=s["out"])
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits

def _grid(y, storage):
    """y rounded to the type's numbers, half to even."""
    if storage == "int8":
        return torch.round(y)
    exponent = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp_min(-6)
    step = torch.exp2(exponent - 3)
    return torch.round(y / step) * step


def _exact_rows(s):
    """q, k, v of the new tokens after norms and rotation, [tokens, heads, entries] in float64."""
    case = s["case"]
    q_heads, k_heads, v_heads, dim, vdim, _ = _sizes(case)
    x = s["qkv"].double()
    tokens = x.shape[0]
    q = x[:, :q_heads * dim]
    k = x[:, q_heads * dim:(q_heads + k_heads) * dim]
    v = x[:, (q_heads + k_heads) * dim:].reshape(tokens, v_heads, vdim)
    rows = []
    for part, heads, weight in ((q, q_heads, s["q_norm"]), (k, k_heads, s["k_norm"])):
        if case["norm"] == "per_head":
            part = part.reshape(tokens, heads, dim)
        if case["norm"] != "none":
            part = part / torch.sqrt((part * part).mean(-1, keepdim=True) + EPS) * weight.double()
        part = part.reshape(tokens, heads, dim).clone()
        for j in range(case["rotary"] // 2):
            one, two = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + case["rotary"] // 2)
            c = s["cos"].double()[s["tok_pos"].long(), j][:, None]
            n = s["sin"].double()[s["tok_pos"].long(), j][:, None]
            a, b = part[:, :, one].clone(), part[:, :, two].clone()
            part[:, :, one], part[:, :, two] = a * c - b * n, b * c + a * n
        rows.append(part)
    return rows[0], rows[1], v


def _exact_put(s, store, scales, x):
    top = x.abs().amax(-1, keepdim=True)
    codes = _grid(x / top.clamp_min(1e-300) * LIMIT[s["case"]["storage"]], s["case"]["storage"])
    pos = s["tok_pos"].long()
    page = s["table"].long()[s["tok_slot"].long(), torch.div(pos, PAGE, rounding_mode="floor")]
    for head in range(x.shape[1]):
        store[page, head, pos % PAGE] = codes[:, head]
        scales[page, head, pos % PAGE] = top[:, head, 0] / LIMIT[s["case"]["storage"]]


def _exact_rows_held(s, name, page, head, place):
    return (s[name].view(torch.uint8)[page, head, place].view(s[name].dtype).double()
            * s[name + "_scale"][page, head, place].double()[:, None])


def _exact_token(s, seq, q, k_of, v_of):
    """The output of one sequence's token, [value heads, group or maps * group, vdim] in float64."""
    case = s["case"]
    q_heads, k_heads, v_heads, dim, vdim, maps = _sizes(case)
    position = _starts(case)[seq]
    first = _first_key(case, position)
    keys = torch.cat([torch.arange(min(case["keep_first"], first), device=DEVICE), torch.arange(first, position + 1, device=DEVICE)])
    page, place = s["table"].long()[s["slot"][seq].long(), keys // PAGE], keys % PAGE
    group = q_heads // k_heads
    out = []
    for h in range(q_heads):
        score = k_of(page, h // group, place) @ q[h] * dim ** -0.5
        if case["softcap"]:
            score = torch.tanh(score / case["softcap"]) * case["softcap"]
        if s["slopes"] is not None:
            score = score - s["slopes"][h].double() * (position - keys)
        if s["sinks"] is not None:
            score = torch.cat([score, s["sinks"][h].double()[None]])
        weight = torch.softmax(score, 0)[:keys.numel()]
        out.append(weight @ v_of(page, h // group // maps, place))
    out = torch.stack(out)
    if maps == 2:
        pairs = out.reshape(v_heads, 2, group, vdim)
        o = pairs[:, 0] - s["lam"].double() * pairs[:, 1]
        out = o / torch.sqrt((o * o).mean(-1, keepdim=True) + DIFF_EPS) * DIFF_FACTOR
    return out.reshape(-1)


def exact(case, seed):
    s = prepare(case, seed)
    q_heads, k_heads, v_heads, dim, vdim, maps = _sizes(case)
    op, out = case["op"], {}
    if op in ("token", "step") and case["seqs"] * q_heads > 1600:
        return None
    codes = {n: s[n] for n in ("k", "v", "k_scale", "v_scale")}
    if op in ("write", "prompt", "step"):
        q, k, v = _exact_rows(s)
        if op == "step":                                    # the new rows beside the others: too many for a copy in 64 bits
            q = q.to(torch.bfloat16)
            fresh = {}
            for name, x in (("k", k), ("v", v)):
                top = x.abs().amax(-1, keepdim=True)
                fresh[name] = (_grid(x / top * LIMIT[case["storage"]], case["storage"]), top / LIMIT[case["storage"]])
            k_new, v_new = (fresh[n][0] * fresh[n][1] for n in ("k", "v"))
            result = []
            for seq in range(case["seqs"]):
                def rows(name, fresh_rows):
                    def of(page, head, place):
                        x = _exact_rows_held(s, name, page, head, place)
                        x[-1] = fresh_rows[seq, head]
                        return x
                    return of
                result.append(_exact_token(s, seq, q[seq].double(), rows("k", k_new), rows("v", v_new)))
            return dict(q=None, k=None, v=None, k_scale=None, v_scale=None, out=torch.stack(result))
        store = {n: codes[n].to(torch.float64) for n in codes}
        _exact_put(s, store["k"], store["k_scale"], k)
        _exact_put(s, store["v"], store["v_scale"], v)
        out.update(q=q.reshape(q.shape[0], -1), k_scale=store["k_scale"], v_scale=store["v_scale"])
        if op == "write":
            out.update(k=store["k"], v=store["v"])
    else:
        store = codes
    if op in ("prompt", "read"):
        keys, values = [], []
        for seq, index in _pages_in_sight(case):
            page = int(s["table"][s["slot"][seq].long(), index])
            count = max(0, min(PAGE, _lengths(case)[seq] - index * PAGE))
            k = store["k"][page].double() * store["k_scale"][page].double()[..., None]
            v = store["v"][page].double() * store["v_scale"][page].double()[..., None]
            k[:, count:] = 0.0
            v[:, count:] = 0.0
            keys.append(k)
            values.append(v.transpose(1, 2))
        out.update(keys=torch.stack(keys), values=torch.stack(values))
    if op == "token":
        def rows(name):
            return lambda page, head, place: _exact_rows_held(s, name, page, head, place)
        q = s["q"].double().reshape(case["seqs"], q_heads, dim)
        out["out"] = torch.stack([_exact_token(s, seq, q[seq], rows("k"), rows("v")) for seq in range(case["seqs"])])
    return out
