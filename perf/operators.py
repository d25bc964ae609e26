"""What the operators of token generation are measured on: head norms with the position rotation
(forward and backward), the int8 cache's write and read, and attention over that cache.

``run`` computes them in elementary torch operations, or, with ``own``, through the library's
entry points: ``tgcb.rotary``, ``tgcb.kv_cache`` and ``tgcb.attention.cached_attention``.
"""

import math
import os
import sys

import torch

own = False

EPSILON = 1e-5
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _rotate(name, op, tokens, q_heads, kv_heads, width, rotary, dtype, interleaved=False, far=4096):
    return {"name": name, "op": op, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "width": width, "rotary": rotary,
            "dtype": dtype, "interleaved": interleaved, "far": far}


def _cache(name, batch, new, context, kv_heads, width, page, dtype):
    return {"name": name, "op": "cache", "batch": batch, "new": new, "context": context, "kv_heads": kv_heads, "width": width,
            "page": page, "dtype": dtype}


def _attend(name, batch, new, context, q_heads, kv_heads, width, page, dtype, cap=0.0, tree=False, ragged=False):
    return {"name": name, "op": "attend", "batch": batch, "new": new, "context": context, "q_heads": q_heads, "kv_heads": kv_heads,
            "width": width, "page": page, "dtype": dtype, "cap": cap, "tree": tree, "ragged": ragged}


def listed():
    return [
        # one sequence's next token: the call is its latency
        _rotate("rotate one token", "rotate", 1, 16, 4, 64, 64, "bfloat16"),
        # a prompt of 8192 tokens at once, 32 query heads on 8 key heads
        _rotate("rotate prompt", "rotate", 8192, 32, 8, 128, 128, "bfloat16", far=65536),
        # float32 training tokens, the first half of each head turned, pairs side by side, an odd count
        _rotate("rotate gradient float32", "rotate_grad", 4095, 16, 4, 128, 64, "float32", interleaved=True),
        # a training batch's gradients in 16 bits
        _rotate("rotate gradient", "rotate_grad", 8192, 32, 8, 128, 128, "bfloat16"),
        # a serving batch writes one token per sequence and reads it back
        _cache("cache step", 64, 1, 2000, 8, 128, 64, "bfloat16"),
        # a prompt's keys and values enter the cache and are read back whole, float32
        _cache("cache prompt", 4, 4096, 0, 8, 128, 64, "float32"),
        # one short sequence, one token: latency
        _attend("attend one token", 1, 1, 300, 16, 4, 64, 16, "bfloat16"),
        # a serving batch of sequences of different lengths
        _attend("attend batch", 64, 1, 4096, 32, 8, 128, 64, "bfloat16", ragged=True),
        # a few very long contexts, float32 queries, capped scores
        _attend("attend long float32", 2, 1, 131072, 32, 8, 128, 64, "float32", cap=30.0),
        # the next piece of a prompt behind what the cache holds, an odd number of tokens
        _attend("attend chunk", 2, 509, 4000, 16, 4, 128, 32, "bfloat16"),
        # a small drafted tree for one sequence, capped scores
        _attend("attend tree", 1, 13, 2047, 32, 8, 128, 64, "float16", cap=50.0, tree=True),
        # drafted trees of a batch, different contexts
        _attend("attend trees batch", 32, 31, 8000, 32, 8, 128, 64, "bfloat16", tree=True, ragged=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate_grad", "cache", "attend", "attend", "attend"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128])
    if op in ("rotate", "rotate_grad"):
        width = rng.choice([32, 64, 80, 96, 128, 256])
        rotary = rng.choice([width, width, width // 2])
        most = max(2, 8192 * 40 * 128 // ((q_heads + kv_heads) * width * (2 if dtype == "float32" else 1)))
        return {**_rotate("", op, _spread(rng, 1, min(16384, most)), q_heads, kv_heads, width, rotary, dtype, rng.random() < 0.4,
                          rng.choice([2048, 32768, 1000000])), "name": "drawn"}
    width = rng.choice([32, 64, 128, 128])
    if op == "cache":
        batch = _spread(rng, 1, 64)
        new = _spread(rng, 1, max(2, 16384 * 8 * 128 // (batch * kv_heads * width * (1 if dtype == "float32" else 1))))
        return {**_cache("", batch, min(new, 8192), rng.choice([0, _spread(rng, 1, 4000)]), kv_heads, width, page, dtype), "name": "drawn"}
    kind = rng.choice(["token", "token", "chunk", "tree"])
    new = 1 if kind == "token" else _spread(rng, 2, 400) if kind == "chunk" else rng.randint(2, 64)
    batch = _spread(rng, 1, 64 if kind == "token" else 4 if kind == "chunk" else 16)
    most = 2 * 131072 * 8 * 128 // (batch * kv_heads * width)
    if kind != "token":
        most = min(most, 32 * 31 * 8000 * 32 * 128 // (batch * new * q_heads * width) // 2, 8000)
    context = _spread(rng, 1, max(2, min(131072, most)))
    return {**_attend("", batch, new, context, q_heads, kv_heads, width, page, dtype, rng.choice([0.0, 0.0, 30.0]), kind == "tree",
                      rng.random() < 0.5), "name": "drawn"}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _table(g, batch, positions, page):
    """A page table whose pages lie anywhere in the cache, and how many pages there are."""
    each = -(-positions // page)
    pages = batch * each + 3
    return torch.randperm(pages, generator=g, device="cuda")[:batch * each].to(torch.int32).reshape(batch, each).contiguous(), pages


def prepare(case, seed):
    g, dtype, width = _generator(seed), DTYPES[case["dtype"]], case["width"]
    if case["op"] in ("rotate", "rotate_grad"):
        n, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        qkv = (_normal(g, n, hq + 2 * hk, width) * 1.5).to(dtype)  # a projection's output: queries, keys and values side by side
        half = case["rotary"] // 2
        s = {"case": case, "queries": qkv[:, :hq], "keys": qkv[:, hq:hq + hk],
             "query_gain": (1 + 0.2 * _normal(g, width)).to(dtype), "key_gain": (1 + 0.2 * _normal(g, width)).to(dtype),
             "positions": torch.randint(0, case["far"], (n,), generator=g, device="cuda", dtype=torch.int32),
             "frequencies": 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)}
        if case["op"] == "rotate_grad":
            s["query_grad"], s["key_grad"] = _normal(g, n, hq, width).to(dtype), _normal(g, n, hk, width).to(dtype)
        return s
    batch, new, context, page, hk = case["batch"], case["new"], case["context"], case["page"], case["kv_heads"]
    table, pages = _table(g, batch, context + new, page)
    s = {"case": case, "table": table, "starts": torch.full((batch,), context, device="cuda", dtype=torch.int32),
         "offsets": None, "tokens": batch * new, "longest": context + new}
    for side in ("key", "value"):
        s[side + "_codes"] = (_normal(g, pages, hk, page, width) * 40).round().clamp(-127, 127).to(torch.int8)
        s[side + "_scales"] = (0.5 + torch.rand(pages, hk, page, generator=g, device="cuda")) / 40
    if case["op"] == "cache":
        spread = torch.exp(0.5 * _normal(g, batch * new, hk, 1))  # rows of different sizes
        s["keys"] = (_normal(g, batch * new, hk, width) * spread).to(dtype)
        s["values"] = (_normal(g, batch * new, hk, width) * spread).to(dtype)
        return s
    if case["ragged"]:
        s["starts"] = torch.randint(context // 4, context + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
        if new > 1:
            even = torch.linspace(1, new, batch, device="cuda", dtype=torch.float64).round().to(torch.int32)
            counts = even[torch.randperm(batch, generator=g, device="cuda")]  # spread over [1, new], in any order
            s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0, dtype=torch.int32)])
            s["tokens"] = int(s["offsets"][-1])
    s["queries"] = (_normal(g, s["tokens"], case["q_heads"], width) * 1.5).to(dtype)
    s["scale"] = width ** -0.5
    if case["tree"]:  # token i hangs on a random earlier one; it sees its ancestors and itself
        parent = (torch.rand(s["tokens"], new, generator=g, device="cuda") * torch.arange(new, device="cuda")).long()
        visible = torch.ones(s["tokens"], new, device="cuda", dtype=torch.int64)
        for i in range(1, new):
            above = visible[:, :i].gather(1, parent[:, i:i + 1])[:, 0]
            visible[:, i] = above | (1 << i if i < 63 else -(1 << 63))
        offsets = s["offsets"] if s["offsets"] is not None else torch.arange(batch + 1, device="cuda") * new
        at = torch.arange(s["tokens"], device="cuda")
        owner = torch.searchsorted(offsets[1:].contiguous().to(torch.int64), at, right=True)
        s["visible"] = visible[offsets[owner].long(), at - offsets[owner]].contiguous()  # one tree for each sequence
    return s


def _turn(x, positions, frequencies, interleaved, back=False):
    """The first 2 * len(frequencies) columns of x [tokens, heads, width], turned by position * frequency."""
    half = frequencies.numel()
    angle = positions.double()[:, None, None] * frequencies  # far positions: angles in 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    sin = -sin if back else sin
    out = x.clone()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    u, v = a * cos - b * sin, a * sin + b * cos
    if interleaved:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = u, v
    else:
        out[..., :half], out[..., half:2 * half] = u, v
    return out


def _plain_rotate(s):
    c, done = s["case"], []
    for x, gain in ((s["queries"], s["query_gain"]), (s["keys"], s["key_gain"])):
        f = x.float()
        y = f * ((f * f).mean(-1, keepdim=True) + EPSILON).rsqrt() * gain.float()
        done.append(_turn(y, s["positions"], s["frequencies"], c["interleaved"]).to(x.dtype))
    return tuple(done)


def _plain_rotate_grad(s):
    c, inputs, gains = s["case"], [], []
    for x, gain, grad in ((s["queries"], s["query_gain"], s["query_grad"]), (s["keys"], s["key_gain"], s["key_grad"])):
        f, dy = x.float(), _turn(grad.float(), s["positions"], s["frequencies"], c["interleaved"], back=True)
        r = ((f * f).mean(-1, keepdim=True) + EPSILON).rsqrt()
        gains.append((dy * f * r).double().sum((0, 1)).to(gain.dtype))
        dn = dy * gain.float()
        inputs.append((r * (dn - f * r * r * (dn * f).mean(-1, keepdim=True))).to(x.dtype))
    return (*inputs, *gains)


def _places(s):
    """Page and row of every new token of a cache case."""
    c = s["case"]
    position = s["starts"].long()[:, None] + torch.arange(c["new"], device="cuda")
    page = s["table"].long().gather(1, position // c["page"])
    return page.reshape(-1), (position % c["page"]).reshape(-1)


def _plain_cache(s):
    page, row = _places(s)
    read = []
    for side in ("key", "value"):
        x = s[side + "s"].float()
        largest = x.abs().amax(-1)
        scale = torch.where(largest == 0, 1.0, (largest.double() / 127).float())
        s[side + "_codes"][page, :, row] = (x / scale[..., None]).round().clamp(-128, 127).to(torch.int8)
        s[side + "_scales"][page, :, row] = scale
        read.append((s[side + "_codes"][page, :, row].float() * s[side + "_scales"][page, :, row][..., None]).to(s[side + "s"].dtype))
    return (*read, s["key_scales"], s["value_scales"])


def _plain_attend(s):
    c = s["case"]
    batch, hk, width, length, new = c["batch"], c["kv_heads"], c["width"], s["longest"], c["new"]
    group = c["q_heads"] // hk
    at = torch.arange(length, device="cuda")
    page, row = s["table"].long()[:, at // c["page"]], (at % c["page"]).expand(batch, -1)
    k = s["key_codes"][page, :, row].float() * s["key_scales"][page, :, row][..., None]  # [batch, length, heads, width]
    v = s["value_codes"][page, :, row].float() * s["value_scales"][page, :, row][..., None]
    offsets = s["offsets"].long() if s["offsets"] is not None else torch.arange(batch + 1, device="cuda") * new
    i = torch.arange(new, device="cuda")
    token = (offsets[:-1, None] + i).clamp(max=s["tokens"] - 1)  # [batch, new], past the sequence's own where it has fewer
    q = s["queries"][token].float().reshape(batch, new, hk, group, width).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * new, width)
    score = (q @ k.permute(0, 2, 3, 1)) * s["scale"]
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    since = at - s["starts"].long()[:, None]  # [batch, length]: which new token a place holds, negative before them
    if c["tree"]:
        bits = (s["visible"][token][:, :, None] >> since.clamp(0, 63)[:, None]) & 1
        seen = torch.where(since[:, None] < 0, True, (bits == 1) & (since[:, None] < new))
    else:
        seen = since[:, None] <= i[:, None]
    score = score.reshape(batch, hk, group, new, length).masked_fill(~seen[:, None, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = (p / p.sum(-1, keepdim=True)).reshape(batch, hk, group * new, length)
    out = (p @ v.permute(0, 2, 1, 3)).reshape(batch, hk, group, new, width).permute(0, 3, 1, 2, 4).reshape(batch, new, hk * group, width)
    mine = i < (offsets[1:] - offsets[:-1])[:, None]
    return out[mine].to(s["queries"].dtype)


def _library(s):
    """The handle of a state's cache, which a program makes once."""
    from tgcb import kv_cache

    if "cache" not in s:
        s["cache"] = kv_cache.QuantisedCache.of(s["key_codes"], s["key_scales"], s["value_codes"], s["value_scales"])
    return s["cache"]


def _own_run(s):
    path = os.path.join(os.getcwd(), "tensor-graph-compiler_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from tgcb import attention, rotary

    c = s["case"]
    if c["op"] == "rotate":
        return rotary.norm_rotate(s["queries"], s["keys"], s["query_gain"], s["key_gain"], s["positions"], s["frequencies"],
                                  epsilon=EPSILON, interleaved=c["interleaved"])
    if c["op"] == "rotate_grad":
        return rotary.norm_rotate_backward(s["query_grad"], s["key_grad"], s["queries"], s["keys"], s["query_gain"], s["key_gain"],
                                           s["positions"], s["frequencies"], epsilon=EPSILON, interleaved=c["interleaved"])
    cache = _library(s)
    if c["op"] == "cache":
        cache.append(s["keys"], s["values"], s["table"], s["starts"])
        keys, values = cache.read(s["tokens"], s["table"], s["starts"], dtype=s["keys"].dtype)
        return keys, values, s["key_scales"], s["value_scales"]
    return attention.cached_attention(s["queries"], cache, s["table"], s["starts"], s["offsets"], visible=s.get("visible"),
                                      scale=s["scale"], cap=c["cap"] or None)


def run(state):
    if own:
        return _own_run(state)
    return {"rotate": _plain_rotate, "rotate_grad": _plain_rotate_grad, "cache": _plain_cache, "attend": _plain_attend}[state["case"]["op"]](state)


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    width, hk = case["width"], case["kv_heads"]
    if case["op"] in ("rotate", "rotate_grad"):
        values = case["tokens"] * (case["q_heads"] + hk) * width
        small = case["tokens"] * 4 + case["rotary"] * 4 + 2 * width * size
        if case["op"] == "rotate":
            return {"bytes": 2 * values * size + small, "flops": 9 * values}
        return {"bytes": 3 * values * size + small + 2 * width * size, "flops": 20 * values}
    batch, new, context = case["batch"], case["new"], case["context"]
    if case["op"] == "cache":  # written: rows in, codes and scales out; read back: the reverse
        rows = 2 * batch * new * hk
        return {"bytes": 2 * rows * (width * size + width + 4), "flops": 6 * rows * width}
    # ragged: contexts are spread evenly over [context / 4, context], counts over [1, new]
    held = context * 0.625 if case["ragged"] else context
    tokens = (new + 1) / 2 if case["ragged"] and new > 1 and batch > 1 else 1 if case["ragged"] else new
    rows = batch * tokens * case["q_heads"]
    seen = held + (tokens + 1) / 2
    return {"bytes": int(2 * batch * hk * (held + tokens) * (width + 4) + 2 * rows * width * size), "flops": int(4 * rows * seen * width)}


def _exact_turn(x, angle, interleaved):
    half, out = angle.shape[-1], x.clone()
    z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else torch.complex(x[..., :half], x[..., half:2 * half])
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rotate", "rotate_grad"):
        angle = s["positions"].double()[:, None] * s["frequencies"][None]
        outs, gains = [], []
        for side in ("query", "key"):
            x, gain = s["queries" if side == "query" else "keys"].double(), s[side + "_gain"].double()
            root = (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPSILON).sqrt()
            unit = x / root
            if case["op"] == "rotate":
                outs.append(_exact_turn(unit * gain, angle, case["interleaved"]))
                continue
            dy = _exact_turn(s[side + "_grad"].double(), -angle, case["interleaved"])
            gains.append((dy * unit).sum((0, 1)))
            dunit = dy * gain
            outs.append((dunit - unit * (dunit * unit).mean(-1, keepdim=True)) / root)
        return (*outs, *gains)
    if case["op"] == "cache":
        page, row = _places(s)
        outs, scales = [], []
        for side in ("key", "value"):
            x = s[side + "s"].double()
            scale = (x.abs().amax(-1) / 127).float()
            scale[scale == 0] = 1.0
            codes = torch.round((x / scale.double()[..., None]).float()).clamp(-128, 127)  # the quotient is a float32, ties to even
            outs.append(codes.double() * scale.double()[..., None])
            whole = s[side + "_scales"].double()
            whole[page, :, row] = scale.double()
            scales.append(whole)
        return (*outs, *scales)
    batch, hk, width = case["batch"], case["kv_heads"], case["width"]
    group, starts = case["q_heads"] // hk, s["starts"].tolist()
    offsets = s["offsets"].tolist() if s["offsets"] is not None else [b * case["new"] for b in range(batch + 1)]
    out = torch.empty(s["tokens"], case["q_heads"], width, device="cuda", dtype=torch.float64)
    for b in range(batch):
        first, last = offsets[b], offsets[b + 1]
        n, length = last - first, starts[b] + last - first
        pages = s["table"][b, :-(-length // case["page"])].long()
        for h in range(hk):
            k, v = ((s[side + "_codes"][pages, h].double() * s[side + "_scales"][pages, h].double()[..., None]).reshape(-1, width)[:length]
                    for side in ("key", "value"))
            q = s["queries"][first:last, h * group:(h + 1) * group].double()
            score = torch.einsum("tgw,lw->tgl", q, k) * s["scale"]
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            seen = torch.ones(n, length, device="cuda", dtype=torch.bool)
            if case["tree"]:
                bit = torch.arange(n, device="cuda")
                seen[:, starts[b]:] = (s["visible"][first:last, None] >> bit) & 1 == 1
            else:
                seen = seen.tril(starts[b])
            weight = torch.softmax(score.masked_fill(~seen[:, None], -math.inf), -1)
            out[first:last, h * group:(h + 1) * group] = torch.einsum("tgl,lw->tgw", weight, v)
    return out
