"""Calls of the stand-alone attention operators: attention of whole prompts, and a key/value cache held in 4 bits with what
writes it, reads it back, attends to it and makes it shorter.

A case is a dict of plain values; ``op`` says which operator:

* "prompt": causal attention of packed prompts, query heads in groups that share a key/value head;
* "write": rows of keys and values go into the 4-bit cache and are read back (what the cache holds is what is returned);
* "step": attention of one token per sequence over the 4-bit cache, with or without the running sums of attention weight;
* "evict": the rows with the largest sums, and the most recent ones, move to a shorter cache.

The 4-bit cache: a row is a token's keys (or values) of one head, in groups of 32 dimensions.  A group with the least value lo
and the largest hi has scale = fp16((hi - lo) / 15) and zero = fp16(lo + 8 scale), and an element x has the code
clamp(round((x - zero) / scale) + 8, 0, 15) (half to even; 8 where scale is 0); it stands for zero + scale (code - 8).  The bytes
of a row are two codes each, the lower dimension in the lower half, then scale and zero of every group.  Dimensions that fill the
last group up count as absent (code 8).
"""
from __future__ import annotations

import math

import torch

own = False

# heads, key/value heads and head size of the models that the benchmark and the tests use
HEADS = {"stories15m": (6, 6, 48), "tinyllama-1.1b": (32, 4, 64), "llama-3.2-1b": (32, 8, 64), "llama-3-8b": (32, 8, 128)}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a story prompt of a llama2.c checkpoint: few heads of an odd size, where latency counts
        dict(name="prompt-stories15m", op="prompt", model="stories15m", dtype="f16", lengths="201", behind=0),
        # a page of text as prompt of a medium model
        dict(name="prompt-1b", op="prompt", model="llama-3.2-1b", dtype="f16", lengths="1023", behind=0),
        # the prompts that waited while a batch was decoded, in a buffer of fixed size: one token up to a few pages
        dict(name="prompt-packed", op="prompt", model="tinyllama-1.1b", dtype="bf16", lengths="1,517,47,1500,0,3,260,129,1100,64", behind=29),
        # a long document as prompt of the largest model
        dict(name="prompt-8b-long", op="prompt", model="llama-3-8b", dtype="bf16", lengths="8192", behind=0),
        # one decoded token of a few sequences goes into the cache
        dict(name="write-step", op="write", model="llama-3-8b", dtype="f32", batch=4, capacity=2048, tokens=4),
        # a long prompt goes into the cache, some of its slots being padding
        dict(name="write-prompt", op="write", model="llama-3-8b", dtype="bf16", batch=1, capacity=8192, tokens=8001),
        # a decoded token behind a medium context of one conversation, in FP32 like the activations of the step
        dict(name="step-1b", op="step", model="llama-3.2-1b", dtype="f32", lengths="641", capacity=2048, weights=False),
        # a decoded token behind a long document, with the sums that eviction goes by
        dict(name="step-8b-32k", op="step", model="llama-3-8b", dtype="f16", lengths="32769", capacity=32784, weights=True),
        # a batch of conversations of different age
        dict(name="step-batch", op="step", model="llama-3-8b", dtype="bf16", lengths="8192,1,700,3001,5555,0,64,129,2047,7000,1025,17,4096,333,6021,90",
             capacity=8192, weights=True),
        # the longest context of the largest model
        dict(name="step-8b-128k", op="step", model="llama-3-8b", dtype="f16", lengths="131071", capacity=131072, weights=False),
        # a conversation outgrows its cache: half of it goes
        dict(name="evict-1b", op="evict", model="llama-3.2-1b", lengths="2048", capacity=2048, keep=1024, recent=64),
        # long documents are cut to what their sums say matters
        dict(name="evict-8b-32k", op="evict", model="llama-3-8b", lengths="32768,20011", capacity=32768, keep=12000, recent=256),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "write", "step", "step", "evict"])
    model = rng.choice(["stories15m", "tinyllama-1.1b", "llama-3.2-1b", "llama-3-8b"])
    case = dict(op=op, model=model)
    if op == "prompt":
        n = rng.choice([1, 1, 2, 5, 12])
        top = {1: 6000, 2: 4000, 5: 1600, 12: 650}[n]
        lengths = [_log_int(rng, 1, top) for _ in range(n)]
        if n == 1 or rng.random() < 0.5:
            lengths[0] = _log_int(rng, 200, top)
        return dict(case, dtype=rng.choice(["f16", "bf16"]), lengths=",".join(map(str, lengths)), behind=rng.choice([0, 0, 1, 100]))
    if op == "write":
        batch = rng.choice([1, 1, 3, 16])
        capacity = 4 * _log_int(rng, 64, 2000 // (1 if batch < 16 else 4))
        return dict(case, dtype=rng.choice(["f32", "f16", "bf16"]), batch=batch, capacity=capacity, tokens=_log_int(rng, 1, min(7000, batch * capacity)))
    batch = rng.choice([1, 1, 2, 9])
    top = {1: 60000, 2: 20000, 9: 5000}[batch]
    lengths = [_log_int(rng, 1, top) for _ in range(batch)]
    lengths[0] = _log_int(rng, 300, top)
    capacity = 4 * ((max(lengths) + 3) // 4 + rng.choice([0, 1, 50]))
    case["lengths"], case["capacity"] = ",".join(map(str, lengths)), capacity
    if op == "step":
        return dict(case, dtype=rng.choice(["f32", "f16", "bf16"]), weights=rng.random() < 0.5)
    keep = min(rng.randint(1, max(lengths)), 12000)
    return dict(case, keep=keep, recent=rng.randint(0, min(keep, 300)))


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _row_bytes(size):
    return 20 * -(-size // GROUP)


# ------------------------------------------------------------------ the 4-bit cache in torch operations

def _pack(x):
    """Rows of the cache for values [..., size], as the module's text defines them, in 64 bits (codes next to a border)."""
    size = x.shape[-1]
    groups = -(-size // GROUP)
    fill = groups * GROUP - size
    x = torch.nan_to_num(x.double(), 0.0, 65504.0, -65504.0).clamp(-65504.0, 65504.0)
    lo = torch.nn.functional.pad(x, (0, fill), value=math.inf).unflatten(-1, (groups, GROUP)).amin(-1)
    hi = torch.nn.functional.pad(x, (0, fill), value=-math.inf).unflatten(-1, (groups, GROUP)).amax(-1)
    scale = ((hi - lo) / 15).half()
    zero = (lo + 8 * scale.double()).half()
    s, z = scale.double().unsqueeze(-1), zero.double().unsqueeze(-1)
    v = torch.nn.functional.pad(x, (0, fill)).unflatten(-1, (groups, GROUP))
    code = torch.where(s > 0, torch.round((v - z) / torch.where(s > 0, s, 1.0)) + 8, 8.0).clamp(0, 15).flatten(-2).to(torch.uint8)
    if fill:
        code[..., size:] = 8
    both = code.unflatten(-1, (-1, 2))
    params = torch.stack([scale, zero], -1).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat([both[..., 0] | (both[..., 1] << 4), params], -1)


def _unpack(rows, size, dtype):
    groups = -(-size // GROUP)
    codes = rows[..., :groups * GROUP // 2]
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (groups, GROUP)).to(dtype)
    params = rows[..., groups * GROUP // 2:].contiguous().view(torch.float16).to(dtype).unflatten(-1, (groups, 2))
    return (params[..., 1:] + params[..., :1] * (codes - 8)).flatten(-2)[..., :size]


# ------------------------------------------------------------------ inputs

def _generator(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 16 + stream)
    return g


def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def _keys(shape, g):
    """Keys have channels that stand out; their sizes are alike for all tokens."""
    channel = torch.exp(0.5 * _normal(shape[-1:], g))
    return _normal(shape, g) * channel


def _cache(shape, g, keys):
    return _pack(_keys(shape, g) if keys else _normal(shape, g) * 0.5)


def prepare(case, seed):
    heads, kv, size = HEADS[case["model"]]
    g = _generator(seed, 0)
    s = dict(op=case["op"], heads=heads, kv=kv, size=size, scale=size ** -0.5)
    if case["op"] == "write":
        dt, n = DTYPES[case["dtype"]], case["tokens"]
        shape = (case["batch"], kv, case["capacity"], _row_bytes(size))
        s["k"], s["v"] = _keys((n, kv, size), g).to(dt), (_normal((n, kv, size), g) * 0.5).to(dt)
        slots = torch.randperm(case["batch"] * case["capacity"], device="cuda", generator=g)[:n]
        if n > 1000:  # a prompt's rows lie behind one another; a portion of fixed size ends with padding
            slots = slots.sort().values
            slots[-7:] = -1
        s["slots"] = slots
        s["k_cache"], s["v_cache"] = (torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2))
        s["k_back"], s["v_back"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    lengths = _lengths(case)
    if case["op"] == "prompt":
        dt, total = DTYPES[case["dtype"]], sum(lengths) + case["behind"]
        s["q"], s["k"] = _keys((total, heads, size), g).to(dt), _normal((total, kv, size), g, dt)
        s["v"] = _normal((total, kv, size), g, dt)
        s["offsets"] = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
        s["out"] = torch.zeros_like(s["q"])
        return s
    cap, batch = case["capacity"], len(lengths)
    s["lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["k_cache"], s["v_cache"] = (_cache((batch, kv, cap, size), g, keys) for keys in (True, False))
    # sums of attention weight: a few rows have most of it
    sums = torch.exp(2.0 * _normal((batch, kv, cap), g)) / cap
    if case["op"] == "step":
        dt = DTYPES[case["dtype"]]
        s["q"] = _normal((batch, heads, size), g, dt)
        s["out"] = torch.zeros_like(s["q"])
        s["sums"], s["sums_out"] = (sums, torch.zeros_like(sums)) if case["weights"] else (None, None)
        return s
    s["sums"], s["keep"], s["recent"] = sums, case["keep"], case["recent"]
    shape = (batch, kv, -(-case["keep"] // 4) * 4)
    s["k_out"], s["v_out"] = (torch.zeros(shape + (_row_bytes(size),), dtype=torch.uint8, device="cuda") for _ in range(2))
    s["sums_out"] = torch.zeros(shape, device="cuda")
    s["kept"] = torch.full((batch, kv, case["keep"]), -1, dtype=torch.int32, device="cuda")
    s["lens_out"] = torch.zeros(batch, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return (_own if own else _plain)[s["op"]](s)


def _own_prompt(s):
    from lighterpp_b200 import ops
    ops.cuda_prompt_attention(s["out"], s["q"], s["k"], s["v"], s["offsets"], s["scale"])
    return s["out"]


def _own_write(s):
    from lighterpp_b200 import ops
    ops.cuda_kv4_write(s["k_cache"], s["v_cache"], s["k"], s["v"], s["slots"])
    ops.cuda_kv4_read(s["k_back"], s["v_back"], s["k_cache"], s["v_cache"], s["slots"])
    return s["k_back"], s["v_back"]


def _own_step(s):
    from lighterpp_b200 import ops
    ops.cuda_kv4_attention(s["out"], s["q"], s["k_cache"], s["v_cache"], s["lens"], s["scale"], s["sums"], s["sums_out"])
    return s["out"], s["sums_out"]


def _own_evict(s):
    from lighterpp_b200 import ops
    ops.cuda_kv4_evict(s["k_out"], s["v_out"], s["sums_out"], s["kept"], s["lens_out"], s["k_cache"], s["v_cache"], s["sums"], s["lens"], s["keep"],
                       s["recent"])
    return s["k_out"], s["v_out"], s["sums_out"], s["kept"], s["lens_out"]


def _plain_prompt(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    total = q.shape[0]
    at = torch.arange(total, device="cuda")
    sequence = torch.searchsorted(s["offsets"], at, right=True)
    visible = (sequence[:, None] == sequence[None, :]) & (at[None, :] <= at[:, None])
    q = q.unflatten(1, (s["kv"], -1)).permute(1, 2, 0, 3)  # key/value head, head of the group, token, dimension
    scores = torch.matmul(q, k.permute(1, 2, 0).unsqueeze(1)).mul_(s["scale"]).masked_fill_(~visible, -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = torch.matmul(scores, v.transpose(0, 1).unsqueeze(1)) / scores.sum(-1, keepdim=True)
    out = out.permute(2, 0, 1, 3).flatten(1, 2).to(s["out"].dtype)
    return torch.where((at < s["offsets"][-1])[:, None, None], out, s["out"])


def _plain_write(s):
    return _written(s["k_cache"], s["k"], s["k_back"], s["slots"]), _written(s["v_cache"], s["v"], s["v_back"], s["slots"])


def _written(cache, x, back, slots):
    """What a cache holds of ``x`` after the write, in ``back`` where a token has no slot."""
    rows = cache.transpose(1, 2).flatten(0, 1)  # slot, key/value head, bytes
    rows = torch.cat([rows, rows[:1]])  # tokens without a slot go behind the last one
    rows[torch.where(slots >= 0, slots, rows.shape[0] - 1)] = _pack(x)
    cache.copy_(rows[:-1].unflatten(0, (cache.shape[0], -1)).transpose(1, 2))
    held = _unpack(rows[slots.clamp(min=0)], x.shape[-1], torch.float32).to(x.dtype)
    return torch.where((slots >= 0)[:, None, None], held, back)


def _plain_step(s):
    k, v = (_unpack(s[c], s["size"], torch.float32) for c in ("k_cache", "v_cache"))
    q = s["q"].float().unflatten(1, (s["kv"], -1))
    inside = torch.arange(k.shape[2], device="cuda") < s["lens"][:, None]
    scores = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    scores = torch.where(inside[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = torch.matmul(p, v).flatten(1, 2).to(s["out"].dtype)
    if s["sums"] is None:
        return out, None
    return out, torch.where(inside[:, None], s["sums"] + p.sum(2), s["sums_out"])


def _plain_evict(s):
    cap, keep = s["sums"].shape[2], s["keep"]
    at = torch.arange(cap, device="cuda")
    lens = s["lens"].long()
    new = lens.clamp(max=keep)
    inside, recent = at < lens[:, None], at >= (lens - s["recent"])[:, None]
    rank = torch.where(recent[:, None], math.inf, s["sums"]).masked_fill(~inside[:, None], -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]  # the lowest row first among equals
    valid = torch.arange(order.shape[-1], device="cuda") < new[:, None]
    order = torch.where(valid[:, None], order, cap).sort(dim=-1).values
    rows = order.clamp(max=cap - 1)
    return (_moved(s["k_cache"], s["k_out"], rows, valid), _moved(s["v_cache"], s["v_out"], rows, valid), _moved(s["sums"], s["sums_out"], rows, valid),
            _moved(at.to(torch.int32).expand(s["sums"].shape), s["kept"], rows, valid), new.to(torch.int32))


def _moved(x, into, rows, valid):
    """``into`` with the named rows of ``x`` [batch, key/value head, row, ...] at its beginning where they are valid."""
    tail = (1,) * (x.dim() - 3)
    rows, valid = rows.view(rows.shape + tail).expand(rows.shape + x.shape[3:]), valid[:, None].view((valid.shape[0], 1, -1) + tail)
    into = into.clone()
    n = rows.shape[2]
    into[:, :, :n] = torch.where(valid, torch.gather(x, 2, rows), into[:, :, :n])
    return into


_own = {"prompt": _own_prompt, "write": _own_write, "step": _own_step, "evict": _own_evict}
_plain = {"prompt": _plain_prompt, "write": _plain_write, "step": _plain_step, "evict": _plain_evict}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    heads, kv, size = HEADS[case["model"]]
    row = _row_bytes(size)
    if case["op"] == "write":
        element = 4 if case["dtype"] == "f32" else 2
        n = case["tokens"]
        return {"bytes": 2 * n * kv * (2 * size * element + 2 * row) + 16 * n, "flops": 2 * n * kv * size * 8}
    lengths = _lengths(case)
    if case["op"] == "prompt":
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        return {"bytes": sum(lengths) * size * 2 * (2 * heads + 2 * kv), "flops": 4 * size * heads * pairs}
    if case["op"] == "step":
        element = 4 if case["dtype"] == "f32" else 2
        total = sum(lengths)
        return {"bytes": total * kv * (2 * row + (8 if case["weights"] else 0)) + 2 * len(lengths) * heads * size * element,
                "flops": 4 * size * heads * total}
    moved = sum(min(n, case["keep"]) for n in lengths)
    return {"bytes": kv * (sum(lengths) * 4 + moved * (4 * row + 8)), "flops": kv * sum(lengths)}


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":
        out = s["out"].double()
        group, first = s["heads"] // s["kv"], 0
        for n in _lengths(case):
            for h in range(s["heads"]):
                q, k, v = (s[x][first:first + n, i].double() for x, i in (("q", h), ("k", h // group), ("v", h // group)))
                a = (q @ k.T) * s["scale"]
                a += torch.full_like(a, -math.inf).triu(1)
                out[first:first + n, h] = torch.softmax(a, -1) @ v
            first += n
        return out
    if case["op"] == "write":
        return tuple(torch.where((s["slots"] >= 0)[:, None, None], _held(s[x]), 0.0) for x in ("k", "v"))
    if case["op"] == "step":
        out, sums = s["out"].double(), None if s["sums"] is None else s["sums_out"].double()
        group = s["heads"] // s["kv"]
        for b, n in enumerate(_lengths(case)):
            for h in range(s["kv"] if n else 0):
                k, v = (_values(s[c][b, h, :n], s["size"]) for c in ("k_cache", "v_cache"))
                p = torch.softmax(s["q"][b, h * group:(h + 1) * group].double() @ k.T * s["scale"], -1)
                out[b, h * group:(h + 1) * group] = p @ v
                if sums is not None:
                    sums[b, h, :n] = s["sums"][b, h, :n].double() + p.sum(0)
        return out, sums
    sums = s["sums_out"].double()
    for b, n in enumerate(_lengths(case)):
        for h in range(s["kv"]):
            w = s["sums"][b, h, :n].tolist()
            old = max(0, n - s["recent"])  # rows before this one are kept by their sums
            some = sorted(range(old), key=lambda i: (-w[i], i))[:max(0, min(n, s["keep"]) - (n - old))]
            kept = sorted(some) + list(range(old, n))
            sums[b, h, :len(kept)] = torch.tensor([w[i] for i in kept], dtype=torch.float64)
    return None, None, sums, None, None  # the rest is moved as it is


def _held(x):
    """What the cache holds of values [..., size]: group by group, from the definition."""
    parts = []
    for part in x.double().split(GROUP, -1):
        part = part.clamp(-65504.0, 65504.0)
        lo, hi = part.aminmax(dim=-1, keepdim=True)
        scale = ((hi - lo) / 15).half().double()
        zero = (lo + 8 * scale).half().double()
        steps = torch.where(scale > 0, torch.round((part - zero) / scale.clamp(min=1e-30)), 0.0)
        parts.append(zero + scale * steps.clamp(-8, 7))
    return torch.cat(parts, -1)


def _values(rows, size):
    """Values of rows [n, bytes], byte by byte."""
    half = rows.shape[-1] * 4 // 5
    dims = torch.arange(size, device=rows.device)
    code = (rows[:, dims // 2].long() >> (4 * (dims % 2))) & 15
    pairs = rows[:, half:].contiguous().view(torch.float16).double()
    return pairs[:, dims // GROUP * 2 + 1] + pairs[:, dims // GROUP * 2] * (code - 8)
