"""What the rotary positions and the packed causal attention of ``agentgarten_b200.ops`` are measured on.

``run`` makes one pass: with ``own`` through the framework's operators, without it through elementary
torch operations in 32 bits.  ``exact`` gives the same outputs from the definitions in 64 bits.

Rotary positions turn the pair ``(a, b)`` of frequency slot ``j`` of a token by the angle ``position *
inverse_j``.  Packed attention is causal softmax attention over sequences laid out back to back, with
grouped key heads; the queries of a sequence are the last rows of its keys.
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One new token of a served prompt: 32 query and 8 key heads of 128; all latency.
        dict(name="rotary token", op="rotary", mode="apply", sequences=1, longest=1, shortest=1, pick=1, heads=32,
             kv_heads=8, dim=128, turned=128, interleaved=False, scaling="none", axes=1, type="bf16"),
        # Eight prompts of up to 514 tokens (the text tower's bucket) packed back to back.
        dict(name="rotary prompts", op="rotary", mode="apply", sequences=8, longest=514, shortest=40, pick=2, heads=32,
             kv_heads=8, dim=128, turned=128, interleaved=False, scaling="linear", axes=1, type="bf16"),
        # One very long prompt whose positions go beyond the trained range: half of every head turned, neighbours paired.
        dict(name="rotary long", op="rotary", mode="apply", sequences=1, longest=65537, shortest=65537, pick=3, heads=32,
             kv_heads=8, dim=128, turned=64, interleaved=True, scaling="yarn", axes=1, type="bf16"),
        # A training step over video tokens with (time, row, column) positions: values and their gradients.
        dict(name="rotary train", op="rotary", mode="train", sequences=1, longest=8190, shortest=8190, pick=4, heads=32,
             kv_heads=8, dim=128, turned=128, interleaved=False, scaling="none", axes=3, type="bf16"),
        # One short prompt: the smallest call of the attention.
        dict(name="prompt short", op="attention", mode="prompt", sequences=1, longest=17, shortest=17, pick=1, heads=32,
             kv_heads=8, dim=128, past=0, type="bf16"),
        # A batch of prompts of very different lengths, up to the text tower's bucket.
        dict(name="prompt batch", op="attention", mode="prompt", sequences=16, longest=514, shortest=11, pick=2, heads=32,
             kv_heads=8, dim=128, past=0, type="bf16"),
        # One long prompt: all matrix products.
        dict(name="prompt long", op="attention", mode="prompt", sequences=1, longest=16384, shortest=16384, pick=3,
             heads=32, kv_heads=8, dim=128, past=0, type="bf16"),
        # A training step of the text tower over packed prompts of middle lengths.
        dict(name="train packed", op="attention", mode="train", sequences=6, longest=2045, shortest=150, pick=4, heads=32,
             kv_heads=8, dim=128, past=0, type="bf16"),
        # The same for a small tower with heads of 64 in half precision.
        dict(name="train small heads", op="attention", mode="train", sequences=3, longest=1000, shortest=90, pick=5,
             heads=8, kv_heads=4, dim=64, past=0, type="fp16"),
        # One token for each of 24 running prompts against their caches, which have room for more.
        dict(name="token batch", op="attention", mode="token", sequences=24, longest=8191, shortest=60, pick=6, heads=32,
             kv_heads=8, dim=128, past=1, type="bf16"),
        # One token of one prompt with a very long cache.
        dict(name="token long", op="attention", mode="token", sequences=1, longest=131071, shortest=131071, pick=7,
             heads=32, kv_heads=8, dim=128, past=1, type="bf16"),
        # Prompts that go on behind a cached part: a few hundred new rows against thousands of keys.
        dict(name="continued prompts", op="attention", mode="continue", sequences=3, longest=301, shortest=5, pick=8,
             heads=32, kv_heads=8, dim=128, past=9000, type="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is even over the range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    pick = rng.randrange(1 << 30)
    if rng.random() < 0.33:
        heads, kv_heads = rng.choice([(32, 8), (4, 2), (16, 16), (8, 1), (12, 4)])
        dim = rng.choice([128, 128, 64, 96, 80])
        total = _spread(rng, 1, 24000)
        sequences = _spread(rng, 1, max(1, min(32, total)))
        longest = max(1, total // sequences)
        axes = rng.choice([1, 1, 3])
        return dict(op="rotary", mode=rng.choice(["apply", "train"]), sequences=sequences, longest=longest,
                    shortest=_spread(rng, 1, longest), pick=pick, heads=heads, kv_heads=kv_heads, dim=dim,
                    turned=dim if axes == 3 else rng.choice([dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), axes=axes,
                    type=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (4, 2), (16, 16), (8, 1), (12, 4)])
    dim = rng.choice([128, 128, 64, 96, 80])
    mode = rng.choice(["prompt", "train", "token", "continue"])
    if mode == "token":
        sequences = _spread(rng, 1, 64)
        longest, past = _spread(rng, 1, 131072 // sequences), 1
    elif mode == "continue":
        sequences = _spread(rng, 1, 8)
        longest, past = _spread(rng, 2, 400), _spread(rng, 1, 24000 // sequences)
    else:
        total = _spread(rng, 2, 12000 if mode == "prompt" else 6000)
        sequences = _spread(rng, 1, max(1, min(48, total // 2)))
        longest, past = max(1, total // sequences), 0
    return dict(op="attention", mode=mode, sequences=sequences, longest=longest, shortest=_spread(rng, 1, longest),
                pick=pick, heads=heads, kv_heads=kv_heads, dim=dim, past=past, type=rng.choice(["bf16", "bf16", "fp16"]))


def _lengths(case):
    """(query rows, keys) of every sequence: logarithms even over the case's range, the last one the longest."""
    rng = random.Random(case["pick"])
    new = [_spread(rng, case["shortest"], case["longest"]) for _ in range(case["sequences"] - 1)] + [case["longest"]]
    if case["op"] == "rotary" or case["mode"] in ("prompt", "train"):
        return new, new
    if case["mode"] == "token":
        return [1] * len(new), new
    return new, [n + _spread(rng, max(1, case["past"] // 8), case["past"]) for n in new]


def work(case):
    new, keys = _lengths(case)
    size = 4 if case["type"] == "fp32" else 2
    query = sum(new) * case["heads"] * case["dim"] * size
    if case["op"] == "rotary":
        key = sum(new) * case["kv_heads"] * case["dim"] * size
        passes = 2 if case["mode"] == "train" else 1
        pairs = sum(new) * (case["heads"] + case["kv_heads"]) * case["turned"] // 2
        return {"bytes": passes * 2 * (query + key) + 4 * case["axes"] * sum(new), "flops": passes * 6 * pairs}
    key = sum(keys) * case["kv_heads"] * case["dim"] * size
    pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(new, keys))
    if case["mode"] == "train":  # q, k, v, the output's gradient; the output and three gradients
        return {"bytes": 4 * query + 4 * key, "flops": 12 * case["dim"] * case["heads"] * pairs}
    return {"bytes": 2 * query + 2 * key, "flops": 4 * case["dim"] * case["heads"] * pairs}


# ------------------------------------------------------------------------------------------ state
THETA = 5_000_000.0
TRAINED = 4096      # positions seen in training, for the scaled frequencies
FACTOR = 8.0
SECTIONS = (24, 20, 20)


def _axis_of_slot(slots):
    """Which of (time, row, column) turns each slot: every third slot is a row's or a column's while that axis has any left."""
    share = [s * slots // 64 for s in SECTIONS]
    return [j % 3 if j % 3 and j < 3 * share[j % 3] else 0 for j in range(slots)]


def _offsets(lengths, device):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = TYPES[case["type"]]
    new, keys = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def values(rows, count):
        return torch.randn(rows, count, dim, device=device, generator=g).to(dtype)

    state = {"case": case}
    if case["op"] == "rotary":
        state["query"], state["key"] = values(sum(new), heads), values(sum(new), kv_heads)
        if case["axes"] == 3:  # frames of 30 x 52 patches at 24/16 positions a frame, behind a prompt
            token = torch.arange(sum(new), device=device)
            grid = torch.stack((token // 1560 * 1.5 + 15000 + 77, token % 1560 // 52, token % 52), dim=-1)
            state["positions"] = grid.float()
        else:
            rows = [torch.arange(n, device=device, dtype=torch.int32) for n in new]
            state["positions"] = torch.cat(rows) + (4093 if sum(new) == 1 else 0)
        if case["mode"] == "train":
            state["grads"] = values(sum(new), heads), values(sum(new), kv_heads)
        if own:
            from agentgarten_b200 import ops

            sections = None if case["axes"] == 1 else tuple(s * (case["turned"] // 2) // 64 for s in SECTIONS)
            state["frequencies"] = ops.rotary_frequencies(
                case["turned"], THETA, scaling=None if case["scaling"] == "none" else case["scaling"], factor=FACTOR,
                trained_positions=TRAINED, sections=sections, device=device)
        if own and case["mode"] == "train":
            state["query"].requires_grad_()
            state["key"].requires_grad_()
        return state
    state["query"] = values(sum(new), heads)
    if case["mode"] == "token":  # a cache with room behind every sequence
        room = case["longest"] + 8 + case["longest"] // 16
        state["key"], state["value"] = values(room * len(new), kv_heads), values(room * len(new), kv_heads)
        state["k_offsets"] = torch.arange(0, room * len(new) + 1, room, dtype=torch.int32, device=device)
        state["k_lengths"] = torch.tensor(keys, dtype=torch.int32, device=device)
    else:
        state["key"], state["value"] = values(sum(keys), kv_heads), values(sum(keys), kv_heads)
        state["k_offsets"], state["k_lengths"] = _offsets(keys, device), None
    state["q_offsets"] = _offsets(new, device)
    if case["mode"] == "train":
        state["grad"] = values(sum(new), heads)
        if own:
            for name in ("query", "key", "value"):
                state[name].requires_grad_()
    return state


def _spans(case):
    """(first query row, rows, first key row, keys) of every sequence."""
    new, keys = _lengths(case)
    room = case["longest"] + 8 + case["longest"] // 16 if case["mode"] == "token" else None
    spans, q, k = [], 0, 0
    for index, (n, m) in enumerate(zip(new, keys)):
        spans.append((q, n, k if room is None else index * room, m))
        q, k = q + n, k + m
    return spans


# ------------------------------------------------------------------------------------ plain form
def _inverse(case):
    """(radians a position of every slot in 64 bits, amplitude)"""
    slots = case["turned"] // 2
    slot = torch.arange(slots, dtype=torch.float64, device="cuda")
    theta, scaling = THETA, case["scaling"]
    if scaling == "ntk":
        theta = THETA * FACTOR ** (case["turned"] / (case["turned"] - 2))
    inverse = theta ** (-slot / slots)
    if scaling == "linear":
        return inverse / FACTOR, 1.0
    if scaling != "yarn":
        return inverse, 1.0

    def slot_of(turns):
        return slots * math.log(TRAINED / (turns * 2 * math.pi)) / math.log(THETA)

    low, high = max(0, math.floor(slot_of(32.0))), min(2 * slots - 1, math.ceil(slot_of(1.0)))
    kept = 1 - ((slot - low) / max(high - low, 1e-3)).clamp(0, 1)
    return inverse * kept + inverse / FACTOR * (1 - kept), 0.1 * math.log(FACTOR) + 1.0


def _angles(case, positions):
    inverse, amplitude = _inverse(case)
    if positions.dim() == 2:
        positions = positions[:, torch.tensor(_axis_of_slot(case["turned"] // 2), device=positions.device)]
    else:
        positions = positions[:, None]
    return positions.double() * inverse, amplitude


def _turn(case, x, cos, sin):
    """One tensor turned in 32 bits and rounded once."""
    slots = case["turned"] // 2
    head = x[..., : 2 * slots].float()
    if case["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = head[..., :slots], head[..., slots:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((turned.to(x.dtype), x[..., 2 * slots:]), dim=-1)


def _plain_rotary(state):
    case = state["case"]
    angle, amplitude = _angles(case, state["positions"])
    cos = (torch.cos(angle) * amplitude).float()[:, None]
    sin = (torch.sin(angle) * amplitude).float()[:, None]
    out = [_turn(case, state["query"], cos, sin), _turn(case, state["key"], cos, sin)]
    if case["mode"] == "train":  # the gradient of a turn is the turn back
        out += [_turn(case, grad, cos, -sin) for grad in state["grads"]]
    return out


def _plain_attention(state):
    case = state["case"]
    query, key, value = state["query"], state["key"], state["value"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, scale, train = heads // kv_heads, dim ** -0.5, case["mode"] == "train"
    out = torch.empty_like(query)
    if train:
        grads = [torch.empty_like(query), torch.empty_like(key), torch.empty_like(value)]
    for q0, rows, k0, keys in _spans(case):
        k = key[k0: k0 + keys].float().transpose(0, 1)                      # [Hkv, keys, D]
        v = value[k0: k0 + keys].float().transpose(0, 1)
        if train:
            dk, dv = torch.zeros_like(k), torch.zeros_like(v)
        block = max(1, min(rows, (1 << 28) // (heads * max(keys, 1))))
        for first in range(0, rows, block):
            n = min(block, rows - first)
            last = min(keys, first + n + keys - rows)                       # keys that the block sees
            q = query[q0 + first: q0 + first + n].float().view(n, kv_heads, group, dim).permute(1, 2, 0, 3)
            s = torch.matmul(q, k[:, None, :last].transpose(-1, -2)) * scale   # [Hkv, group, n, last]
            row = torch.arange(first, first + n, device=q.device)[:, None] + (keys - rows)
            hidden = torch.arange(last, device=q.device)[None] > row
            s.masked_fill_(hidden, float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = torch.matmul(p, v[:, None, :last])
            out[q0 + first: q0 + first + n] = o.permute(2, 0, 1, 3).reshape(n, heads, dim).to(out.dtype)
            if train:
                do = state["grad"][q0 + first: q0 + first + n].float().view(n, kv_heads, group, dim).permute(1, 2, 0, 3)
                dv[:, :last] += torch.matmul(p.transpose(-1, -2), do).sum(1)
                ds = p * (torch.matmul(do, v[:, None, :last].transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)) * scale
                dk[:, :last] += torch.matmul(ds.transpose(-1, -2), q).sum(1)
                dq = torch.matmul(ds, k[:, None, :last])
                grads[0][q0 + first: q0 + first + n] = dq.permute(2, 0, 1, 3).reshape(n, heads, dim).to(out.dtype)
        if train:
            grads[1][k0: k0 + keys] = dk.transpose(0, 1).to(out.dtype)
            grads[2][k0: k0 + keys] = dv.transpose(0, 1).to(out.dtype)
    return [out, *grads] if train else [out]


def run(state):
    case = state["case"]
    if not own:
        return _plain_rotary(state) if case["op"] == "rotary" else _plain_attention(state)
    from agentgarten_b200 import ops

    if case["op"] == "rotary":
        turned = ops.rotary_embed(state["query"], state["key"], state["positions"], state["frequencies"],
                                  interleaved=case["interleaved"])
        if case["mode"] != "train":
            return list(turned)
        grads = torch.autograd.grad(turned, (state["query"], state["key"]), state["grads"])
        return [t.detach() for t in turned] + list(grads)
    out = ops.packed_attention(state["query"], state["key"], state["value"], state["q_offsets"], state["k_offsets"],
                               k_lengths=state["k_lengths"])
    if case["mode"] != "train":
        return [out]
    return [out.detach(), *torch.autograd.grad(out, (state["query"], state["key"], state["value"]), state["grad"])]


# ---------------------------------------------------------------------------------------- exact
def _exact_rotary(state):
    """Pairs as complex numbers, multiplied by amplitude * exp(i angle)."""
    case = state["case"]
    angle, amplitude = _angles(case, state["positions"])
    wheel = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    slots = case["turned"] // 2
    where = torch.arange(slots, device=angle.device)
    first, second = (2 * where, 2 * where + 1) if case["interleaved"] else (where, where + slots)

    def turned(x, by):
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = [turned(state["query"], wheel), turned(state["key"], wheel)]
    if case["mode"] == "train":
        out += [turned(grad, wheel.conj()) for grad in state["grads"]]
    return out


def _exact_attention(state):
    """Head by head in 64 bits; the gradients through torch's own differentiation of the definition."""
    case = state["case"]
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    train = case["mode"] == "train"
    query, key, value = (state[name] for name in ("query", "key", "value"))
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (query, key, value)] if train else []
    for q0, rows, k0, keys in _spans(case):
        late = torch.arange(keys, device=query.device)[None] - torch.arange(rows, device=query.device)[:, None] > keys - rows
        for h in range(heads):
            q, k, v = (t.double().detach() for t in (query[q0: q0 + rows, h], key[k0: k0 + keys, h // group],
                                                     value[k0: k0 + keys, h // group]))
            with torch.set_grad_enabled(train):
                for t in (q, k, v):
                    t.requires_grad_(train)
                s = q @ k.t() / math.sqrt(case["dim"])
                o = torch.softmax(s.masked_fill(late, -math.inf), dim=-1) @ v
            out[q0: q0 + rows, h] = o.detach()
            if train:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["grad"][q0: q0 + rows, h].double())
                grads[0][q0: q0 + rows, h] = dq
                grads[1][k0: k0 + keys, h // group] += dk
                grads[2][k0: k0 + keys, h // group] += dv
    return [out, *grads]


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_rotary(state) if case["op"] == "rotary" else _exact_attention(state)
