"""The operators of the answering side of a vision-language decoder: what each is measured on, its plain form and its definition.

  rotary   rotary positions with several axes (time, height, width) applied to queries and keys; "train" adds both gradients
  pages    block tables, lengths and the slot map of the next tokens, for a cache in pages
  append   keys and values of new tokens written to a cache held in 4 bits, and read back from it
  attend   attention of the newest tokens over that cache: grouped heads, requests of different lengths, pages in any order

The cache is one uint8 tensor [pages, kv heads, page_size / 16, slice].  A slice holds 16 tokens of one head: the codes of the
keys, their group parameters, the codes of the values, their group parameters.  A group is `group` neighbouring channels of
a token; its parameters are a step and a lowest value of the tensors' type, and code n stands for lowest + n * step.

Run from the repository's root.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAGE = 64


def _ops():
    package = os.path.join(os.getcwd(), "pyramid-sparse-attention_b200")
    if package not in sys.path:
        sys.path.insert(1, package)
    from psa_b200 import ops
    return ops


# ---------------------------------------------------------------- cases

def listed():
    vl = dict(heads=28, kv_heads=4, dim=128, batch=1, sections="16,24,24", layout="half", per_axis=False, theta=1e6, train=False)
    video = dict(batch=1, layout="pairs", per_axis=True, theta=1e4)
    return [
        # one new token of a vision-language decoder behind a long prompt: latency
        dict(vl, name="rotary one token", op="rotary", dtype="bf16", tokens=1, text=0, far=120000),
        # its prompt: text, a video's grid, text
        dict(vl, name="rotary prompt", op="rotary", dtype="bf16", tokens=32768, text=500, far=0),
        # self-attention of a video model, token-major projections, neighbouring channels paired (832 x 480, 81 frames)
        dict(video, name="rotary video", op="rotary", dtype="f16", heads=12, kv_heads=12, dim=128, sections="22,21,21", tokens=32760,
             text=0, far=0, train=False),
        # a training step of a video model with 226 text tokens in front (720 x 480, 49 frames), forward and both gradients
        dict(video, name="rotary video train", op="rotary", dtype="bf16", heads=48, kv_heads=48, dim=64, sections="8,12,12",
             tokens=17776, text=226, far=0, train=True),
        # the next token of every request of a running batch
        dict(name="pages next token", op="pages", requests=64, tokens=1, least=1, shortest=100, longest=30000, width=512),
        # new requests: their whole prompts, of very different lengths
        dict(name="pages prompts", op="pages", requests=250, tokens=8192, least=9, shortest=0, longest=0, width=2048),
        # keys and values of the next token of every request
        dict(name="append next token", op="append", dtype="bf16", batch=16, tokens=1, kv_heads=4, dim=128, group=32),
        # keys and values of a prompt
        dict(name="append prompt", op="append", dtype="f16", batch=1, tokens=32761, kv_heads=4, dim=128, group=64),
        # a short conversation, one token: latency
        dict(name="attend one short", op="attend", dtype="bf16", batch=1, tokens=1, heads=28, kv_heads=4, dim=128, group=32,
             shortest=500, longest=500),
        # requests of very different lengths, every head with keys of its own
        dict(name="attend ragged", op="attend", dtype="f16", batch=33, tokens=1, heads=16, kv_heads=16, dim=64, group=64,
             shortest=17, longest=16384),
        # long contexts, one token of each request
        dict(name="attend long", op="attend", dtype="bf16", batch=8, tokens=1, heads=28, kv_heads=4, dim=128, group=32,
             shortest=131000, longest=131071),
        # several tokens of each request at once (drafted tokens to be checked)
        dict(name="attend several tokens", op="attend", dtype="bf16", batch=5, tokens=6, heads=28, kv_heads=4, dim=128, group=64,
             shortest=9000, longest=32760),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "pages", "append", "append", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "rotary":
        layout = rng.choice(["half", "pairs"])
        dim = rng.choice([64, 128])
        sections = rng.choice({64: ["8,12,12", "32", "10,11,11"], 128: ["16,24,24", "22,21,21", "64", "32,32"]}[dim])
        kv = rng.choice([1, 2, 4, 8, 12])
        heads = kv * rng.choice([1, 2, 4, 7])
        batch = rng.choice([1, 1, 2, 3])
        train = rng.random() < 0.4
        most = 1.6e8 / (batch * (heads + kv) * dim * (2 if train else 1))
        return dict(op=op, dtype=rng.choice([dtype, dtype, "f32"]), heads=heads, kv_heads=kv, dim=dim, batch=batch, sections=sections,
                    layout=layout, per_axis=layout == "pairs", theta=rng.choice([1e4, 1e6]), tokens=_log(rng, 1, min(60000, most)),
                    text=rng.choice([0, 3, 77]), far=rng.choice([0, 0, 50000, 1000000]), train=train)
    if op == "pages":
        tokens = _log(rng, 1, 8192)
        return dict(op=op, requests=_log(rng, 1, 300), tokens=tokens, least=rng.randint(0, tokens), shortest=_log(rng, 1, 90),
                    longest=_log(rng, 90, 20000), width=rng.choice([511, 1024, 2000]))
    dim = rng.choice([64, 128])
    group = rng.choice([32, 64] if dim == 64 else [32, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    if op == "append":
        batch = _log(rng, 1, 100)
        return dict(op=op, dtype=dtype, batch=batch, tokens=_log(rng, 1, 1.2e5 / (batch * kv)), kv_heads=kv, dim=dim, group=group)
    batch = _log(rng, 1, 64)
    longest = _log(rng, 20, min(131072, 3e6 / (batch * kv)))
    return dict(op=op, dtype=dtype, batch=batch, tokens=rng.choice([1, 1, 1, 2, 3, 5, 8]), heads=kv * rng.choice([1, 2, 4, 7, 8]), kv_heads=kv,
                dim=dim, group=group, shortest=_log(rng, 8, longest), longest=longest)


def _lengths(case):
    """Context lengths of a case's requests, from the shortest to the longest, spread over their logarithm."""
    n, low, high = case.get("batch", case.get("requests")), case["shortest"], case["longest"]
    if low <= 0:
        return [0] * n
    return [int(round(low * (high / low) ** (i / max(1, n - 1)))) for i in range(n - 1)] + [high]


def _counts(case):
    n, low, high = case["requests"], case["least"], case["tokens"]
    return [int(round(low + (high - low) * i / max(1, n - 1))) for i in range(n - 1)] + [high]


def _slice_bytes(dim, group):
    return 16 * (dim + 8 * (dim // group))


def work(case):
    op = case["op"]
    if op == "rotary":
        values = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"] * (2 if case["train"] else 1)
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * values * size + 12 * case["batch"] * case["tokens"], "flops": 3 * values}
    if op == "pages":
        n = case["requests"]
        return {"bytes": 4 * (2 * n * case["width"] + 4 * n + n * case["tokens"] + sum(_counts(case)) // PAGE), "flops": n * case["tokens"]}
    rows = case["batch"] * case["tokens"] * case["kv_heads"]
    if op == "append":
        return {"bytes": rows * (8 * case["dim"] + 2 * _slice_bytes(case["dim"], case["group"]) // 16), "flops": 8 * rows * case["dim"]}
    context, new = sum(_lengths(case)), case["batch"] * case["tokens"] * case["heads"] * case["dim"]
    return {"bytes": context * case["kv_heads"] * _slice_bytes(case["dim"], case["group"]) // 16 + 4 * new,
            "flops": 4 * context * case["tokens"] * case["heads"] * case["dim"]}


# ---------------------------------------------------------------- inputs

def _positions(case):
    """int32 [axes, batch, tokens].  One axis: a running number.  Several: text, a grid of (time, height, width), text that goes
    on behind it; a video model's text in front stands at the origin and is not turned."""
    axes, batch, n, text = len(case["sections"].split(",")), case["batch"], case["tokens"], case["text"]
    t = torch.arange(n)
    if axes == 1:
        p = t[None]
    else:
        across, down = 52, 30
        at = t - text
        grid = torch.stack([at // (across * down), at // across % down, at % across][:axes])
        if case["per_axis"]:
            p = torch.where(t < text, 0, grid)
        else:
            behind = n - n // 8
            p = torch.where(t < text, t, torch.where(t < behind, text + grid, t - behind + text + max(across, n // (across * down))))
    p = p[:, None, :] + case["far"] + torch.arange(batch)[None, :, None] * (0 if case["per_axis"] else 17)
    return p.to(torch.int32).to(DEVICE)


def _channels(g, dim, spread):
    """Channels of a projection do not have one size: some are a few times the others."""
    return torch.exp(spread * torch.randn(dim, generator=g, device=DEVICE))


def _rows(g, shape, dtype, spread=0.5, offset=0.0):
    scale = _channels(g, shape[-1], spread)
    x = torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=g)
    x *= scale.to(dtype)
    if offset:
        x += (offset * torch.randn(shape[-1], generator=g, device=DEVICE)).to(dtype)
    return x


def _tables(g, lengths, pages, width):
    """Pages of every request in no order; entries that no request has reached say -1."""
    held = (lengths + PAGE - 1) // PAGE
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    first = torch.cumsum(held, 0) - held
    j = torch.arange(width, device=DEVICE)
    table = torch.where(j < held[:, None], order[(first[:, None] + j).clamp(max=pages - 1)], -1)
    return table.to(torch.int32), order[int(held.sum()):]


def _quantised(x, group):
    """Codes (uint8, one a channel), steps and lowest values of x [..., dim]."""
    y = x.float().unflatten(-1, (-1, group))
    low, high = y.amin(-1), y.amax(-1)
    wide = (high - low) / 15
    step = wide.to(x.dtype)
    # towards zero: lowest + 15 * step is never above the highest value
    step = torch.where(step.float() > wide, (step.view(torch.int16) - 1).view(x.dtype), step)
    s = step.float().unsqueeze(-1)
    code = torch.where(s > 0, (y - low.unsqueeze(-1)) / s, torch.zeros_like(y)).round().clamp(0, 15)
    return code.flatten(-2).to(torch.uint8), step, low.to(x.dtype)


def _places(dim, group):
    """Byte offsets within a slice, [16, dim / 2] of the code bytes of keys and of values (two neighbouring channels a byte, the
    first in the low half) and [16, groups] of their parameters (step, then lowest)."""
    t, d = torch.arange(16, device=DEVICE)[:, None], torch.arange(0, dim, 2, device=DEVICE)[None]
    blocks, groups = dim // 32, dim // group
    row = 8 * (t // 8) + 2 * (t % 4) + t // 4 % 2
    k = row * (dim // 2) + (d % 32 // 8 * blocks + d // 32) * 4 + d % 8 // 2
    eighth = d % 32 // 4
    if dim == 128:
        eighth = eighth ^ (t // 2 % 2 * 4)
    v = t * (dim // 2) + (eighth * blocks + d // 32) * 2 + d % 4 // 2
    p = (row * groups + torch.arange(groups, device=DEVICE)[None]) * 4
    half = _slice_bytes(dim, group) // 2
    return k, 8 * dim + p, half + v, half + 8 * dim + p


def _write(data, k, v, slots, group):
    """Rows k, v [batch, kv heads, tokens, dim] into the cache at slots [batch, tokens]."""
    dim, flat, slot = k.shape[-1], data.view(-1), slots.flatten().long()
    base = (slot // PAGE * data.shape[1])[:, None] + torch.arange(data.shape[1], device=DEVICE)
    base = (base * data.shape[2] + (slot % PAGE // 16)[:, None]) * data.shape[3]
    at = _places(dim, group)
    _put(flat, k, base, at[0][slot % 16], at[1][slot % 16], group)
    _put(flat, v, base, at[2][slot % 16], at[3][slot % 16], group)


def _put(flat, x, base, codes_at, params_at, group):
    code, step, low = _quantised(x.transpose(1, 2).flatten(0, 1), group)
    flat[base[..., None] + codes_at[:, None]] = code[..., 0::2] | code[..., 1::2] << 4
    words = torch.stack([step, low], -1).view(torch.uint8)                                      # [rows, kv heads, groups, 4]
    flat[base[..., None, None] + params_at[:, None, :, None] + torch.arange(4, device=DEVICE)] = words


def _slots(table, lengths, tokens):
    """Slots of the last `tokens` tokens of every request."""
    at = lengths[:, None] - tokens + torch.arange(tokens, device=DEVICE)
    return (torch.gather(table, 1, at // PAGE) * PAGE + at % PAGE).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    op = case["op"]
    if op == "pages":
        lengths = torch.tensor(_lengths(case), device=DEVICE, dtype=torch.int32)
        counts = torch.tensor(_counts(case), device=DEVICE, dtype=torch.int32)
        counts = counts[torch.randperm(len(counts), generator=g, device=DEVICE)]
        counts = torch.minimum(counts, case["width"] * PAGE - lengths)
        need = int(((lengths + counts + PAGE - 1) // PAGE).sum())
        table, pool = _tables(g, lengths.long(), need + 37, case["width"])
        return dict(case, table=table, lengths=lengths, counts=counts, pool=pool, free=torch.tensor([len(pool)], dtype=torch.int32, device=DEVICE))
    dtype, batch, n = DTYPES[case["dtype"]], case["batch"], case["tokens"]
    if op == "rotary":
        s = dict(case, positions=_positions(case), sections=tuple(int(x) for x in case["sections"].split(",")))
        # projections are token-major: what an attention layer sees are transposed views
        names = ("q", "k", "dq", "dk") if case["train"] else ("q", "k")
        for name, heads in zip(names, (case["heads"], case["kv_heads"]) * 2):
            s[name] = _rows(g, (batch, n, heads, case["dim"]), dtype, 0.3).transpose(1, 2)
        if case["train"]:
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    kv, dim, group = case["kv_heads"], case["dim"], case["group"]
    context = [n] * batch if op == "append" else _lengths(case)
    context = torch.tensor(context, device=DEVICE)[torch.randperm(batch, generator=g, device=DEVICE)]
    width = (int(context.max()) + PAGE - 1) // PAGE
    pages = int(((context + PAGE - 1) // PAGE).sum()) + 11
    table, _ = _tables(g, context, pages, width)
    data = torch.zeros(pages, kv, PAGE // 16, _slice_bytes(dim, group), dtype=torch.uint8, device=DEVICE)
    lengths = context.to(torch.int32)
    s = dict(case, data=data, table=table, lengths=lengths, dtype=dtype)
    if op == "append":
        s["k"] = _rows(g, (batch, n, kv, dim), dtype, 0.5, 0.5).transpose(1, 2)
        s["v"] = _rows(g, (batch, n, kv, dim), dtype, 0.2).transpose(1, 2)
        s["slots"] = _slots(table, context, n)
        return s
    # the keys' and values' channels are the same for every token of a call, as a layer's are
    ks, vs = _channels(g, dim, 0.4).to(dtype), _channels(g, dim, 0.2).to(dtype)
    bias = (0.5 * torch.randn(dim, generator=g, device=DEVICE)).to(dtype)
    step = max(1, (1 << 20) // kv // PAGE)
    for i in range(0, pages, step):
        m = min(step, pages - i)
        k = torch.empty(1, kv, m * PAGE, dim, dtype=dtype, device=DEVICE).normal_(generator=g) * ks + bias
        v = torch.empty(1, kv, m * PAGE, dim, dtype=dtype, device=DEVICE).normal_(generator=g) * vs
        _write(data[i:i + m], k, v, torch.arange(m * PAGE, device=DEVICE)[None], group)
    s["q"] = (torch.randn(batch, n, case["heads"], dim, generator=g, device=DEVICE) * 1.2).to(dtype).transpose(1, 2)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    return {"rotary": _run_rotary, "pages": _run_pages, "append": _run_append, "attend": _run_attend}[state["op"]](state)


def _run_rotary(s):
    if own:
        q, k = _ops().rotate_axes(s["q"], s["k"], s["positions"], s["sections"], theta=s["theta"], layout=s["layout"], per_axis=s["per_axis"])
        if not s["train"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return q.detach(), k.detach(), dq, dk
    with torch.no_grad():
        cos, sin = _cos_sin(s["positions"], s["sections"], s["theta"], s["per_axis"])
        out = _turned(s["q"], cos, sin, s["layout"]), _turned(s["k"], cos, sin, s["layout"])
        if not s["train"]:
            return out
        # the transposed rotation turns back
        return (*out, _turned(s["dq"], cos, -sin, s["layout"]), _turned(s["dk"], cos, -sin, s["layout"]))


def _cos_sin(positions, sections, theta, per_axis):
    """float32 [batch, 1, tokens, pairs]; the angles in 64 bits: far positions."""
    pairs = sum(sections)
    # the number of a pair, in its section or among all, over how many there are
    size = torch.tensor(sections, dtype=torch.float64)
    within = torch.arange(pairs, dtype=torch.float64)
    if per_axis:
        within = (within - torch.repeat_interleave(torch.cumsum(size, 0) - size, size.long())) / torch.repeat_interleave(size, size.long())
    else:
        within = within / pairs
    freq = (theta ** -within).to(positions.device)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(positions.device)
    angle = positions[axis].permute(1, 2, 0).double() * freq
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _turned(x, cos, sin, layout):
    y = x.float()
    if layout == "half":
        a, b = y.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2).to(x.dtype)


def _run_pages(s):
    if own:
        return _ops().plan_pages(s["table"], s["lengths"], s["counts"], s["pool"], s["free"], PAGE, s["tokens"])
    table, lengths, counts, pool, free = s["table"], s["lengths"], s["counts"], s["pool"], s["free"]
    width = table.shape[1]
    fits = lengths + counts <= width * PAGE
    counts = torch.where(fits, counts, 0)
    held = (lengths + PAGE - 1) // PAGE
    need = (lengths + counts + PAGE - 1) // PAGE - held
    total = torch.cumsum(need, 0)
    served = (need == 0) | (total <= free)
    counts = torch.where(served, counts, 0)
    first = total - need
    need = torch.where(served, need, 0)
    # page j of a request is the next one from the top of the pool
    j = torch.arange(width, device=table.device) - held[:, None]
    fresh = (j >= 0) & (j < need[:, None])
    table = torch.where(fresh, pool[(free - 1 - first[:, None] - j).clamp(0, len(pool) - 1)], table)
    i = torch.arange(s["tokens"], device=table.device)
    at = lengths[:, None] + i
    slots = torch.gather(table, 1, (at // PAGE).clamp(max=width - 1).long()) * PAGE + at % PAGE
    slots = torch.where(i < counts[:, None], slots, -1)
    return table, (lengths + counts).to(torch.int32), (free - need.sum()).to(torch.int32), slots.to(torch.int32)


def _run_append(s):
    if own:
        ops = _ops()
        ops.kv4_append(s["data"], s["k"], s["v"], s["slots"], s["group"])
        return ops.kv4_read(s["data"], s["slots"], s["dim"], s["group"], s["dtype"])
    _write(s["data"], s["k"], s["v"], s["slots"], s["group"])
    dim, group, slots = s["dim"], s["group"], s["slots"].long()
    kv = s["data"].shape[1]
    head = torch.arange(kv, device=slots.device)[None, :, None]
    part = s["data"][(slots // PAGE)[:, None], head, (slots % PAGE // 16)[:, None]]          # [batch, kv heads, tokens, slice]
    at = [p[slots % 16][:, None].expand(-1, kv, -1, -1) for p in _places(dim, group)]
    return (_values(part, at[0], at[1], group, s["dtype"]).to(s["dtype"]), _values(part, at[2], at[3], group, s["dtype"]).to(s["dtype"]))


def _values(part, codes_at, params_at, group, dtype):
    """What rows stand for, in 32 bits: part [..., slice] their slices, codes_at and params_at their bytes in them."""
    byte = torch.gather(part, -1, codes_at)
    code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2).float().unflatten(-1, (-1, group))
    words = torch.gather(part, -1, (params_at[..., None] + torch.arange(4, device=part.device)).flatten(-2))
    step, low = words.view(dtype).float().unflatten(-1, (-1, 2)).unbind(-1)
    return (low[..., None] + code * step[..., None]).flatten(-2)


def _whole(part, codes_at, params_at, group, dtype):
    """The same for whole slices: part [..., slice] -> [..., 16, dim]."""
    byte = part[..., codes_at]
    code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2).float().unflatten(-1, (-1, group))
    words = part[..., params_at[..., None] + torch.arange(4, device=part.device)].contiguous()
    step, low = words.view(dtype).float().unbind(-1)
    return (low[..., None] + code * step[..., None]).flatten(-2)


def _run_attend(s):
    if own:
        return _ops().kv4_attention(s["q"], s["data"], s["table"], s["lengths"], s["group"])
    q, dim = s["q"], s["dim"]
    batch, heads, n, _ = q.shape
    kv = s["data"].shape[1]
    part = s["data"][s["table"].clamp(min=0).long()].transpose(1, 2)                          # [batch, kv heads, pages, 4, slice]
    at = _places(dim, s["group"])
    q = q.float().reshape(batch, kv, heads // kv * n, dim) * dim ** -0.5
    scores = q @ _whole(part, at[0], at[1], s["group"], s["dtype"]).flatten(2, 4).transpose(-1, -2)
    # the i-th of n new tokens stands at length - n + i and sees what is not behind it
    last = s["lengths"][:, None] - n + torch.arange(n, device=q.device)
    seen = torch.arange(scores.shape[-1], device=q.device) <= last[..., None]
    scores = scores.unflatten(2, (-1, n)).masked_fill(~seen[:, None, None], -math.inf).flatten(2, 3)
    weight = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (weight @ _whole(part, at[2], at[3], s["group"], s["dtype"]).flatten(2, 4)) / weight.sum(-1, keepdim=True)
    return out.reshape(batch, heads, n, dim).to(s["dtype"])


# ---------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    if case["op"] == "pages":
        return None
    s = prepare(case, seed)
    if case["op"] == "rotary":
        # pairs as complex numbers, multiplied by exp(i angle)
        angles, pair = [], 0
        for axis, n in enumerate(s["sections"]):
            for j in range(n):
                part = j / n if s["per_axis"] else (pair + j) / sum(s["sections"])
                angles.append(s["positions"][axis].double() * math.exp(-part * math.log(s["theta"])))
            pair += n
        angle = torch.stack(angles, -1)[:, None]
        out, half = [], s["layout"] == "half"
        for name in ("q", "k", "dq", "dk")[:4 if s["train"] else 2]:
            x = s[name].detach().double()
            z = x.unflatten(-1, (2, -1)).transpose(-1, -2) if half else x.unflatten(-1, (-1, 2))
            z = torch.complex(z[..., 0], z[..., 1]) * torch.polar(torch.ones_like(angle), angle if name in "qk" else -angle)
            y = torch.view_as_real(z)
            out.append((y.transpose(-1, -2) if half else y).flatten(-2))
        return out
    if case["op"] == "append":
        return [_stored(s[x], s["group"]) for x in ("k", "v")]
    # request by request, head by head, with logarithms of sums
    q, data, dim = s["q"].double(), s["data"], s["dim"]
    batch, heads, n, _ = q.shape
    kv = data.shape[1]
    places = _places(dim, s["group"])
    out = torch.empty_like(q)
    for b, length in enumerate(s["lengths"].tolist()):
        pages = data[s["table"][b, :(length + PAGE - 1) // PAGE].long()]
        place = torch.arange(length, device=q.device)
        for h in range(kv):
            x = pages[:, h].reshape(-1, data.shape[3])
            rows = []
            for codes, params in (places[:2], places[2:]):
                byte = x[:, codes].int()
                value = torch.empty(*byte.shape[:2], dim, dtype=torch.float64, device=q.device)
                value[..., 0::2], value[..., 1::2] = byte % 16, byte // 16
                words = [(x[:, params + i].int() + 256 * x[:, params + i + 1].int()).to(torch.int16).view(s["dtype"]) for i in (0, 2)]
                step, low = (w.double().repeat_interleave(s["group"], -1) for w in words)
                rows.append((low + step * value).reshape(-1, dim)[:length])
            mine = slice(h * (heads // kv), (h + 1) * (heads // kv))
            score = torch.einsum("gid,td->git", q[b, mine], rows[0]) / math.sqrt(dim)
            score = torch.where(place > length - n + torch.arange(n, device=q.device)[:, None], -math.inf, score)
            out[b, mine] = torch.einsum("git,td->gid", torch.exp(score - torch.logsumexp(score, -1, keepdim=True)), rows[1])
    return out


def _stored(x, group):
    """Which of the 16 values of its group's scale each value is stored as.  The step is a number of the tensor's type, cut off
    and not rounded; a value halfway between two codes takes the even one."""
    y = x.double().unflatten(-1, (-1, group))
    low = y.min(-1, keepdim=True).values
    step = (y.max(-1, keepdim=True).values - low) / 15
    bits, least = (8, -125) if x.dtype == torch.bfloat16 else (11, -13)
    exponent = torch.frexp(step)[1].clamp(min=least)                                           # subnormal numbers below it
    grid = torch.exp2((exponent - bits).double())
    step = torch.floor(step / grid) * grid
    code = torch.where(step > 0, torch.round((y - low) / torch.where(step > 0, step, 1.0)), 0.0)
    return (low + torch.clamp(code, max=15.0) * step).flatten(-2)
