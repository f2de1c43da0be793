"""The attention half of a decoder layer around a paged key/value cache, case by case.

Three operators: ``rotary`` (rotary position embedding of queries and keys, with its gradient),
``append`` (new keys and values written into the pages of a cache, the rotation applied on the
way) and ``attend`` (causal attention of each sequence's newest tokens over its pages).

Each case can be computed in plain form (elementary torch operations in fp32, angles in fp64)
or, with ``own`` set, by the framework's kernels.  ``exact`` evaluates the definitions in fp64.
"""
import importlib
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------- cases
def _rotary(name, batch, length, first, q_heads, k_heads, dim, rot, layout, scaling, factor, dtype, backward):
    return {"name": name, "op": "rotary", "batch": batch, "length": length, "first": first, "q_heads": q_heads,
            "k_heads": k_heads, "dim": dim, "rot": rot, "layout": layout, "scaling": scaling, "factor": factor,
            "dtype": dtype, "backward": backward}


def _append(name, seqs, new, context, ragged, q_heads, k_heads, dim, rot, layout, page, dtype):
    return {"name": name, "op": "append", "seqs": seqs, "new": new, "context": context, "ragged": ragged,
            "mixed": False, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "rot": rot, "layout": layout,
            "page": page, "dtype": dtype}


def _attend(name, seqs, new, context, ragged, mixed, q_heads, k_heads, dim, page, dtype):
    return {"name": name, "op": "attend", "seqs": seqs, "new": new, "context": context, "ragged": ragged,
            "mixed": mixed, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "page": page, "dtype": dtype}


def listed():
    return [
        # one decode step of a batch of 16 in the 12-head decoder: pure latency
        _rotary("rotary step", 16, 1, 500, 12, 12, 128, 128, "half", "none", 1.0, "bf16", False),
        # a training step of the 12-head model: 8 sequences of 2048, gradients of q and k
        _rotary("rotary training", 8, 2048, 0, 12, 12, 128, 128, "half", "none", 1.0, "bf16", True),
        # a long document, half of each head rotated, grouped heads, positions far past the trained length
        _rotary("rotary far", 1, 32768, 100003, 32, 8, 128, 64, "interleaved", "yarn", 8.0, "fp16", False),
        # one decode step of a batch of 16 in the 12-head decoder (prompt 512, up to 128 new tokens)
        _append("append step", 16, 1, 639, True, 12, 12, 128, 128, "half", 16, "bf16"),
        # 16 prompts of 512 tokens into an empty cache
        _append("append prompts", 16, 512, 0, False, 12, 12, 128, 128, "half", 16, "bf16"),
        # ragged chunks behind ragged contexts, grouped heads, larger pages, fp16
        _append("append chunks", 12, 2011, 5003, True, 32, 8, 128, 64, "interleaved", 64, "fp16"),
        # one sequence of the 12-head decoder answering: the smallest call, pure latency
        _attend("attend one", 1, 1, 639, False, False, 12, 12, 128, 16, "bf16"),
        # a serving batch, one new token each, ragged contexts
        _attend("attend batch", 64, 1, 8191, True, False, 32, 8, 128, 16, "bf16"),
        # two very long conversations, one new token each: few rows, a long axis
        _attend("attend long", 2, 1, 131070, False, False, 32, 8, 128, 64, "bf16"),
        # a few proposed tokens for each sequence checked at once, 64-wide heads, fp16
        _attend("attend verify", 24, 5, 4001, True, False, 16, 4, 64, 32, "fp16"),
        # 16 prompts of 512 tokens from the start
        _attend("attend prompts", 16, 512, 0, False, False, 12, 12, 128, 16, "bf16"),
        # a chunk of 2048 tokens of a long document over all that came before it
        _attend("attend chunk", 1, 2048, 32768, False, False, 32, 8, 128, 128, "bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


_HEADS = [(12, 12), (32, 8), (16, 4), (16, 2), (8, 1), (6, 2), (20, 4), (4, 4), (15, 3)]


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend"])
    q_heads, k_heads = rng.choice(_HEADS)
    dim = rng.choice([64, 128, 128])
    layout = rng.choice(["half", "interleaved"])
    rot = rng.choice([dim, dim, dim // 2, dim // 4])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rotary":
        batch, length = _log(rng, 1, 32), _log(rng, 1, 32768)
        while batch * length * (q_heads + k_heads) * dim > 130_000_000:
            batch, length = max(1, batch // 2), length * 3 // 4
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        c = _rotary("", batch, length, _log(rng, 1, 200000) - 1, q_heads, k_heads, dim, rot, layout, scaling,
                    1.0 if scaling == "none" else float(rng.choice([2, 4, 8])),
                    rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5)
    else:
        kind = rng.choice(["step", "verify", "prompt", "chunk", "mixed"])
        page = rng.choice([16, 32, 64, 128, 256])
        if kind == "step":
            seqs, new, context = _log(rng, 1, 128), 1, _log(rng, 1, 100000) - 1
        elif kind == "verify":
            seqs, new, context = _log(rng, 1, 64), rng.randint(2, 8), _log(rng, 1, 20000)
        elif kind == "prompt":
            seqs, new, context = _log(rng, 1, 16), _log(rng, 2, 4096), 0
        else:
            seqs, new, context = _log(rng, 1, 16), _log(rng, 9, 2048), _log(rng, 1, 32768)
        # cache values and (padded) score values stay below those of the largest listed cases
        while seqs * (new + context + page) * k_heads * dim > 250_000_000 or \
                seqs * new * (new + context) * q_heads > (150_000_000 if op == "append" else 2_000_000_000):
            if seqs > 1:
                seqs = max(1, seqs * 2 // 3)
            elif context:
                context = context * 2 // 3
            else:
                new = max(1, new * 2 // 3)
        ragged = rng.random() < 0.75
        if op == "append":
            c = _append("", seqs, new, context, ragged, q_heads, k_heads, dim, rot, layout, page, dtype)
            c["mixed"] = kind == "mixed"
        else:
            c = _attend("", seqs, new, context, ragged, kind == "mixed", q_heads, k_heads, dim, page, dtype)
    del c["name"]
    return c


def _lengths(case):
    """New tokens and cached length (new ones included) of each sequence; they follow from the case alone."""
    r = random.Random("%d %d %d" % (case["seqs"], case["new"], case["context"]))
    new, total = [], []
    for i in range(case["seqs"]):
        n, c = case["new"], case["context"]
        if case["ragged"] and i:
            n, c = r.randint(1, n), r.randint(0, c)
        if case["mixed"] and i % 2:
            n = 1
        new.append(n)
        total.append(n + c)
    return new, total


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    hq, hk, d = case["q_heads"], case["k_heads"], case["dim"]
    if case["op"] == "rotary":
        tokens = case["batch"] * case["length"]
        passes = 2 if case["backward"] else 1
        return {"bytes": passes * tokens * (2 * (hq + hk) * d * size + 8),
                "flops": passes * tokens * (hq + hk) * case["rot"] * 3}
    new, total = _lengths(case)
    tables = 4 * (2 * case["seqs"] + 1) + 4 * sum(-(-t // case["page"]) for t in total)
    if case["op"] == "append":
        tokens = sum(new)
        return {"bytes": 2 * tokens * (hq + 2 * hk) * d * size + tables, "flops": tokens * (hq + hk) * case["rot"] * 3}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return {"bytes": 2 * sum(new) * hq * d * size + 2 * sum(total) * hk * d * size + tables,
            "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------------- inputs
def _turns(rot, scaling, factor, base=10000.0, trained=4096):
    """Turns per position of each rotated pair (fp64) and the factor on rotated values."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if scaling == "linear":
        f = f / factor
    gain = 1.0
    if scaling == "yarn":
        at = lambda beta: rot * math.log(trained / (beta * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        keep = 1 - ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    return f / (2 * math.pi), gain


def _package():
    return importlib.import_module("prune_path_openpangu-embedded-1b_b200")


def _embedding(case):
    kind = case.get("scaling", "none")
    scaling = None if kind == "none" else {"type": kind, "factor": case["factor"]}
    if kind == "yarn":
        scaling["original_length"] = 4096
    return _package().rotary.RotaryEmbedding(case["dim"], rotary_dim=case["rot"], layout=case["layout"], scaling=scaling)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    hq, hk, d = case["q_heads"], case["k_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    s = {"case": case}
    if case["op"] != "attend":
        turns, s["gain"] = _turns(case["rot"], case.get("scaling", "none"), case.get("factor", 1.0))
        s["turns"] = turns.to(dev)
        if own:
            s["embedding"] = _embedding(case)
    if case["op"] == "rotary":
        b, n = case["batch"], case["length"]
        # queries and keys are parts of one projection's output, as a layer has them
        qk = normal(b, n, hq + hk, d)
        s["q"], s["k"] = qk[:, :, :hq], qk[:, :, hq:]
        start = torch.randint(0, 64, (b, 1), generator=g, device=dev)
        s["positions"] = case["first"] + start + torch.arange(n, device=dev)
        if case["backward"]:
            s["dq"], s["dk"] = normal(b, n, hq, d), normal(b, n, hk, d)
            if own:
                s["q"], s["k"] = s["q"].requires_grad_(), s["k"].requires_grad_()
        return s
    new, total = _lengths(case)
    page = case["page"]
    need = [-(-t // page) for t in total]
    pages, widest = sum(need), max(need)
    # pages are handed out in no order; what lies behind a sequence's last page in its row is -1
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    count = torch.tensor(need, device=dev)
    column = torch.arange(widest, device=dev)
    at = (count.cumsum(0) - count)[:, None] + column
    s["table"] = torch.where(column < count[:, None], order[at.clamp(max=pages - 1)], -1).to(torch.int32)
    s["starts"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    s["lengths"] = torch.tensor(total, device=dev, dtype=torch.int32)
    s["most_new"], s["most_length"] = max(new), max(total)
    tokens = sum(new)
    s["k_pages"], s["v_pages"] = normal(pages, hk, page, d), normal(pages, hk, page, d)
    if own:
        s["cache"] = _package().kvcache.PagedKVCache.from_tensors(s["k_pages"], s["v_pages"])
    if case["op"] == "append":
        qkv = normal(tokens, hq + 2 * hk, d)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    else:
        s["q"] = normal(tokens, hq, d) * 2
    return s


# ---------------------------------------------------------------------------------- plain forms
def _turned(x, cos, sin, rot, layout):
    """x [..., heads, dim] in fp32 with its first `rot` values rotated; cos, sin [..., 1, rot / 2]."""
    r, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = r[..., 0::2], r[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _angles(s, positions):
    turn = positions.double()[..., None, None] * s["turns"]
    angle = (turn - turn.round()) * (2 * math.pi)
    return (angle.cos() * s["gain"]).float(), (angle.sin() * s["gain"]).float()


def _places(s):
    """Sequence, place within its new tokens and position of every new token."""
    token = torch.arange(s["q"].shape[0], device=s["q"].device, dtype=torch.int32)
    seq = torch.searchsorted(s["starts"], token, right=True) - 1
    nth = token - s["starts"][seq]
    return seq, nth.long(), (s["lengths"][seq] - (s["starts"][seq + 1] - s["starts"][seq]) + nth).long()


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angles(s, s["positions"])
    dt = s["q"].dtype
    out = {n: _turned(s[n].float(), cos, sin, c["rot"], c["layout"]).to(dt) for n in ("q", "k")}
    if c["backward"]:
        out |= {n: _turned(s[n].float(), cos, -sin, c["rot"], c["layout"]).to(dt) for n in ("dq", "dk")}
    return out


def _plain_append(s):
    c = s["case"]
    seq, _, pos = _places(s)
    cos, sin = _angles(s, pos)
    q, k = (_turned(s[n].float(), cos, sin, c["rot"], c["layout"]).to(s["q"].dtype) for n in ("q", "k"))
    page = s["table"][seq, pos // c["page"]].long()
    s["k_pages"][page, :, pos % c["page"]] = k
    s["v_pages"][page, :, pos % c["page"]] = s["v"]
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attend(s):
    c = s["case"]
    hq, hk, d = c["q_heads"], c["k_heads"], c["dim"]
    seqs, most, group = c["seqs"], s["most_new"], hq // hk
    dev = s["q"].device
    # the new tokens of all sequences padded to the longest: [seqs, kv heads, group * most, dim]
    nth = torch.arange(most, device=dev)
    row = (s["starts"][:-1, None] + nth).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][row].float().view(seqs, most, hk, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * most, d)
    new = s["starts"][1:] - s["starts"][:-1]
    pos = (s["lengths"] - new)[:, None] + nth
    # each sequence's pages side by side: [seqs, kv heads, keys, dim]
    table = s["table"].clamp(min=0).long()
    k, v = (s[n][table].transpose(1, 2).reshape(seqs, hk, -1, d).float() for n in ("k_pages", "v_pages"))
    key = torch.arange(k.shape[2], device=dev)
    score = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(seqs, hk, group, most, -1)
    score.masked_fill_((key > pos[:, :, None])[:, None, None], -math.inf)
    weight = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(seqs, hk, group * most, -1) @ v).view(seqs, hk, group, most, d) / total
    seq, nth, _ = _places(s)
    return out.permute(0, 3, 1, 2, 4)[seq, nth].reshape(-1, hq, d).to(s["q"].dtype)


# ---------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[c["op"]](s)
    if c["op"] == "rotary":
        if not c["backward"]:
            q, k = s["embedding"](s["q"], s["k"], s["positions"])
            return {"q": q, "k": k}
        q, k = s["embedding"](s["q"], s["k"], s["positions"])
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    cache = s["cache"]
    if c["op"] == "append":
        q = cache.append(s["q"], s["k"], s["v"], s["starts"], s["lengths"], s["table"], rotary=s["embedding"])
        return {"q": q, "k_pages": cache.k, "v_pages": cache.v}
    return cache.attend(s["q"], s["starts"], s["lengths"], s["table"], max_new=s["most_new"], max_length=s["most_length"])


# ---------------------------------------------------------------------------------- definitions in 64 bits
def _complex_turn(x, positions, s, sign):
    """The rotation as a product of complex numbers in fp64."""
    c = s["case"]
    rot, layout = c["rot"], c["layout"]
    phase = torch.remainder(positions.double()[..., None] * s["turns"], 1.0) * (2 * math.pi * sign)
    unit = torch.polar(torch.full_like(phase, s["gain"]), phase)[..., None, :]
    y = x.double().clone()
    if layout == "half":
        z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * unit
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    else:
        z = torch.complex(y[..., 0:rot:2], y[..., 1:rot:2]) * unit
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        out = {n: _complex_turn(s[n], s["positions"], s, 1) for n in ("q", "k")}
        if case["backward"]:
            out |= {n: _complex_turn(s[n], s["positions"], s, -1) for n in ("dq", "dk")}
        return out
    new, total = _lengths(case)
    size, d = case["page"], case["dim"]
    hk, group = case["k_heads"], case["q_heads"] // case["k_heads"]
    dev = s["q"].device
    if case["op"] == "append":
        q = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        t = 0
        for b, (n, length) in enumerate(zip(new, total)):
            pos = torch.arange(length - n, length, device=dev)
            part = slice(t, t + n)
            q[part] = _complex_turn(s["q"][part], pos, s, 1)
            page = s["table"][b].long()[pos // size]
            k_pages[page, :, pos % size] = _complex_turn(s["k"][part], pos, s, 1)
            v_pages[page, :, pos % size] = s["v"][part].double()
            t += n
        return {"q": q, "k_pages": k_pages, "v_pages": v_pages}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
    t = 0
    for b, (n, length) in enumerate(zip(new, total)):
        pages = s["table"][b, :-(-length // size)].long()
        future = torch.ones(n, length, dtype=torch.bool, device=dev).triu(length - n + 1)
        for h in range(hk):
            k, v = (s[x][pages, h].reshape(-1, d)[:length].double() for x in ("k_pages", "v_pages"))
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][t:t + n, j].double() @ k.T / math.sqrt(d)).masked_fill(future, -math.inf)
                out[t:t + n, j] = torch.softmax(score, -1) @ v
        t += n
    return out
