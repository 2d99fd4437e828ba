"""The serving steps around a paged 8-bit KV cache, as cases to measure: rotary positions, appending keys and values to
the cache, attention over it, and causal attention over packed prompts.

`run(state)` computes a case in plain torch operations, or, with `own` set, through larder_b200.ops. The cases are
listed in `listed()`; `draw(rng)` gives others of the same ranges.

The cache: pages [num_pages, 2 (K, V), Hkv, page, D] in float8 e4m3, scales [num_pages, 2, Hkv] fp32 (powers of two, one
for each page and head of K and of V), table [B, max_pages] int32 (a sequence's pages in order). A held value is
code * scale.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODE_MAX = 448.0  # the largest e4m3 value


def listed():
    return [
        # one decode step's queries of 16 sequences deep in a stretched context: latency
        {"name": "rope_decode", "op": "rope", "B": 16, "T": 1, "H": 32, "D": 128, "R": 128, "layout": "half",
         "dtype": "bf16", "far": 131072, "factor": 4.0, "inverse": False},
        # the queries of a whole packed prompt, adjacent pairs rotated
        {"name": "rope_prompt", "op": "rope", "B": 1, "T": 8192, "H": 32, "D": 128, "R": 128, "layout": "interleaved",
         "dtype": "f16", "far": 8192, "factor": 1.0, "inverse": False},
        # the gradient of a partial rotation (a quarter of wide heads), an odd number of fp32 rows
        {"name": "rope_gradient", "op": "rope", "B": 3, "T": 1667, "H": 16, "D": 256, "R": 64, "layout": "half",
         "dtype": "f32", "far": 32768, "factor": 1.0, "inverse": True},
        # one new token for each of 64 running sequences
        {"name": "append_decode", "op": "append", "B": 64, "T": 1, "Hkv": 8, "D": 128, "R": 128, "layout": "half",
         "page": 64, "dtype": "bf16", "before": 4096, "packed": False},
        # packed prompts of uneven lengths going into fresh and half-filled pages
        {"name": "append_prompts", "op": "append", "B": 9, "T": 4100, "Hkv": 4, "D": 128, "R": 64,
         "layout": "interleaved", "page": 16, "dtype": "bf16", "before": 70, "packed": True},
        # a long prompt's keys and values in one call
        {"name": "append_long", "op": "append", "B": 2, "T": 16384, "Hkv": 8, "D": 128, "R": 128, "layout": "half",
         "page": 64, "dtype": "f16", "before": 0, "packed": False},
        # one short conversation: latency
        {"name": "attend_one", "op": "attend", "B": 1, "T": 1, "Hq": 32, "Hkv": 8, "D": 128, "N": 777, "page": 16,
         "dtype": "bf16"},
        # a batch of sequences of uneven lengths, one token each
        {"name": "attend_batch", "op": "attend", "B": 16, "T": 1, "Hq": 32, "Hkv": 4, "D": 128, "N": 8192, "page": 64,
         "dtype": "bf16"},
        # four draft tokens checked at once with wide heads and many query heads a KV head
        {"name": "attend_verify", "op": "attend", "B": 4, "T": 4, "Hq": 24, "Hkv": 2, "D": 256, "N": 16390, "page": 32,
         "dtype": "f16"},
        # many long sequences: a full card's decode step
        {"name": "attend_full", "op": "attend", "B": 64, "T": 1, "Hq": 32, "Hkv": 8, "D": 128, "N": 32768, "page": 128,
         "dtype": "bf16"},
        # many short prompts admitted together
        {"name": "prompts_short", "op": "prompts", "S": 33, "T": 4001, "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16"},
        # a few long prompts with wide heads
        {"name": "prompts_long", "op": "prompts", "S": 3, "T": 12288, "Hq": 16, "Hkv": 2, "D": 256, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "prompts"])
    D = rng.choice([64, 128, 256])
    half = rng.choice(["bf16", "f16"])
    if op == "rope":
        B, T = rng.choice([(_log(rng, 1, 96), 1), (rng.randint(1, 3), _log(rng, 2, 5000))])
        H = rng.choice([2, 5, 8, 16, 32]) if D < 256 else rng.choice([2, 5, 8, 16])
        return {"op": op, "B": B, "T": T, "H": H, "D": D, "R": rng.choice([D, D // 2, D // 4]),
                "layout": rng.choice(["half", "interleaved"]), "dtype": rng.choice(["bf16", "f16", "f32"]),
                "far": _log(rng, 6000, 500000), "factor": rng.choice([1.0, 4.0]), "inverse": rng.random() < 0.4}
    if op == "append":
        c = {"op": op, "D": D, "R": rng.choice([0, D // 2, D]), "layout": rng.choice(["half", "interleaved"]),
             "Hkv": rng.choice([1, 2, 4, 8]), "page": rng.choice([16, 32, 64, 128]),
             "dtype": rng.choice(["bf16", "f16", "f32"]), "packed": rng.random() < 0.5}
        if rng.random() < 0.4:
            return {**c, "B": _log(rng, 1, 128), "T": 1, "before": _log(rng, 1, 4000), "packed": False}
        return {**c, "B": rng.randint(1, 8), "T": _log(rng, 8, 4000), "before": rng.choice([0, 1, 37, 128])}
    if op == "attend":
        Hkv = rng.choice([1, 2, 4, 8])
        G = rng.choice([1, 3, 4, 8])
        B = _log(rng, 1, 64)
        N = min(_log(rng, 20, 60000), 2_000_000 // B)
        return {"op": op, "B": B, "T": rng.choice([1, 1, 1, 2, 5]), "Hq": G * Hkv, "Hkv": Hkv, "D": D, "N": N,
                "page": rng.choice([16, 32, 64, 128]), "dtype": half}
    Hkv = rng.choice([1, 2, 4])
    G = rng.choice([1, 4, 7, 8]) if D < 256 else rng.choice([1, 4, 8])
    return {"op": op, "S": _log(rng, 1, 60), "T": _log(rng, 100, 6000), "Hq": G * Hkv, "Hkv": Hkv, "D": D,
            "dtype": half}


# ------------------------------------------------------------------------------------------------ lengths of a case


def _cuts(total, parts):
    """`parts` uneven lengths that sum to `total` (some may be 0 where there are more parts than rows)."""
    rng = random.Random(total * 1009 + parts)
    w = [rng.random() ** 2 + 0.02 for _ in range(parts)]
    at = [0]
    for i in range(parts):
        at.append(total if i == parts - 1 else min(total, int(total * sum(w[:i + 1]) / sum(w))))
    return [at[i + 1] - at[i] for i in range(parts)]


def _kept(c):
    """Tokens already in the cache and tokens that come, for each sequence of an append."""
    rng = random.Random(c["B"] * 7919 + c["T"])
    before = [rng.randint(c["before"] // 2, c["before"]) for _ in range(c["B"])]
    return before, _cuts(c["T"], c["B"]) if c["packed"] else [c["T"]] * c["B"]


def _lens(c):
    """Cached keys of each sequence of an attention over the cache, this call's among them."""
    rng = random.Random(c["B"] * 7919 + c["N"])
    return [max(c["T"], c["N"] if b == 0 else rng.randint(c["N"] // 2, c["N"])) for b in range(c["B"])]


def work(c):
    if c["op"] == "rope":
        item = 4 if c["dtype"] == "f32" else 2
        n = c["B"] * c["T"] * c["H"]
        return {"bytes": 2.0 * n * c["D"] * item, "flops": 3.0 * n * c["R"]}
    if c["op"] == "append":
        n = sum(_kept(c)[1]) * c["Hkv"] * c["D"]
        return {"bytes": n * 2.0 * ((4 if c["dtype"] == "f32" else 2) + 1), "flops": 8.0 * n}
    if c["op"] == "attend":
        keys, rows = sum(_lens(c)), c["B"] * c["T"] * c["Hq"]
        return {"bytes": 2.0 * keys * c["Hkv"] * c["D"] + 4.0 * rows * c["D"],
                "flops": 4.0 * keys * c["T"] * c["Hq"] * c["D"]}
    pairs = sum(n * (n + 1) // 2 for n in _cuts(c["T"], c["S"]))
    return {"bytes": 2.0 * c["T"] * c["D"] * (2 * c["Hq"] + 2 * c["Hkv"]), "flops": 4.0 * pairs * c["Hq"] * c["D"]}


# ------------------------------------------------------------------------------------------------ inputs


def _frequencies(R, factor):
    """Angles a position, in radians: the usual base, its low half stretched by `factor` (a long-context scaling)."""
    return [10000.0 ** (-2 * i / R) / (factor if 4 * i >= R else 1.0) for i in range(R // 2)]


def _turns(R, factor, dev):
    """The same as 64-bit fractions of a turn, which a position multiplies exactly."""
    f = [int(round(w / (2 * math.pi) * 2.0 ** 64)) for w in _frequencies(R, factor)]
    return torch.tensor([x - (1 << 64) if x >= 1 << 63 else x for x in f], dtype=torch.int64, device=dev)


def _amp(factor):
    return 1.0 if factor == 1.0 else 0.1 * math.log(factor) + 1.0


def _codes(x):
    """Pages x [..., page, D] fp32 as e4m3 codes and their power-of-two scales [...]."""
    m = x.abs().amax((-2, -1))
    s = torch.where(m > 0, torch.exp2(torch.ceil(torch.log2(m / CODE_MAX))), torch.zeros_like(m))
    s = torch.where(m > s * CODE_MAX, s * 2, s)
    return torch.where(s[..., None, None] > 0, x / s[..., None, None], torch.zeros_like(x)).to(torch.float8_e4m3fn), s


def _cache(gen, dev, lens, page, Hkv, D):
    """A filled cache for sequences of these lengths, its pages in no order."""
    per = [max(1, -(-n // page)) for n in lens]
    num = sum(per) + 3
    order = torch.randperm(num, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(per), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    pages = torch.empty(num, 2, Hkv, page, D, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(num, 2, Hkv, device=dev)
    loud = torch.ones(2, 1, 1, D, device=dev)
    loud[0, :, :, ::37] = 6.0  # a few loud key channels
    step = max(1, (1 << 26) // (2 * Hkv * page * D))
    for i in range(0, num, step):
        x = torch.randn(min(step, num - i), 2, Hkv, page, D, generator=gen, device=dev) * loud
        p, scales[i:i + step] = _codes(x)
        pages.view(torch.uint8)[i:i + step] = p.view(torch.uint8)
    return pages, scales, table


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev).to(dt)

    def rows(B, H, T, D):  # heads-first views of token-major rows, as projections leave them
        return normal(B, T, H, D).transpose(1, 2)

    s = {"op": c["op"]}
    if c["op"] == "rope":
        s["x"] = rows(c["B"], c["H"], c["T"], c["D"])
        first = torch.randint(0, max(1, c["far"] - c["T"] + 1), (c["B"], 1), generator=gen, device=dev)
        s["positions"] = (first + torch.arange(c["T"], device=dev)).to(torch.int32)
        s["turns"], s["amp"] = _turns(c["R"], c["factor"], dev), _amp(c["factor"])
        s["layout"], s["inverse"] = c["layout"], c["inverse"]
    elif c["op"] == "append":
        before, new = _kept(c)
        s["pages"], s["scales"], s["table"] = _cache(gen, dev, [a + b for a, b in zip(before, new)], c["page"],
                                                     c["Hkv"], c["D"])
        B, T = (1, sum(new)) if c["packed"] else (c["B"], c["T"])
        loud = torch.ones(c["D"], device=dev)
        loud[::37] = 6.0
        s["k"] = (rows(B, c["Hkv"], T, c["D"]) * loud.to(dt))
        s["v"] = rows(B, c["Hkv"], T, c["D"])
        s["start"] = torch.tensor(before, dtype=torch.int32, device=dev)
        s["cu"] = None
        if c["packed"]:
            s["cu"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)
        s["longest"] = max(new)
        s["turns"], s["layout"] = (_turns(c["R"], 1.0, dev) if c["R"] else None), c["layout"]
    elif c["op"] == "attend":
        lens = _lens(c)
        s["pages"], s["scales"], s["table"] = _cache(gen, dev, lens, c["page"], c["Hkv"], c["D"])
        s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["q"] = rows(c["B"], c["Hq"], c["T"], c["D"])
        s["scale"] = c["D"] ** -0.5
    else:
        lens = _cuts(c["T"], c["S"])
        s["cu"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)
        s["longest"] = max(lens)
        s["q"] = rows(1, c["Hq"], c["T"], c["D"])
        s["k"], s["v"] = rows(1, c["Hkv"], c["T"], c["D"]), rows(1, c["Hkv"], c["T"], c["D"])
        s["scale"] = c["D"] ** -0.5
    return s


# ------------------------------------------------------------------------------------------------ the operators


def run(s):
    if own:
        from larder_b200 import ops
        if s["op"] == "rope":
            return ops.rope(s["x"], s["positions"], s["turns"], s["layout"], s["amp"], s["inverse"])
        if s["op"] == "append":
            ops.kv8_append(s["pages"], s["scales"], s["k"], s["v"], s["table"], s["start"], cu=s["cu"],
                           turns=s["turns"], layout=s["layout"])
            return {"pages": s["pages"], "scales": s["scales"]}
        if s["op"] == "attend":
            return ops.kv8_attend(s["q"], s["pages"], s["scales"], s["table"], s["kv_len"], s["scale"])
        return ops.attn_packed(s["q"], s["k"], s["v"], s["scale"], s["cu"])
    if s["op"] == "rope":
        amp = s["amp"]
        return _rotate(s["x"].float(), s["positions"], s["turns"], s["layout"], amp, s["inverse"]).to(s["x"].dtype)
    return {"append": _append, "attend": _attend, "prompts": _prompts}[s["op"]](s)


def _rotate(x, positions, turns, layout, amp=1.0, inverse=False):
    """x [B, H, T, D] fp32 with its first 2 len(turns) dims rotated by the positions [B, T]."""
    R = 2 * turns.numel()
    a = (positions.long()[:, None, :, None] * turns).float() * (2 * math.pi / 2.0 ** 64)
    c, n = torch.cos(a) * amp, torch.sin(a) * (-amp if inverse else amp)
    if layout == "half":
        x0, x1 = x[..., :R // 2], x[..., R // 2:R]
        y = torch.cat([x0 * c - x1 * n, x1 * c + x0 * n], -1)
    else:
        x0, x1 = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack([x0 * c - x1 * n, x1 * c + x0 * n], -1).flatten(-2)
    return torch.cat([y, x[..., R:]], -1)


def _append(s):
    pages, scales, table, start = s["pages"], s["scales"], s["table"], s["start"].long()
    page, dev, B = pages.shape[3], pages.device, start.numel()
    k, v = s["k"].float(), s["v"].float()
    if s["cu"] is None:
        first = torch.arange(B, device=dev) * k.shape[2]
        count = torch.full((B,), k.shape[2], device=dev)
        at = start[:, None] + torch.arange(k.shape[2], device=dev)
    else:
        first, count = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
        row = torch.arange(k.shape[2], device=dev)
        seq = torch.bucketize(row, s["cu"][1:].long(), right=True)
        at = (row - first[seq] + start[seq])[None]
    if s["turns"] is not None:
        k = _rotate(k, at, s["turns"], s["layout"])
    rows = torch.stack([k, v], 0).permute(1, 3, 0, 2, 4).flatten(0, 1)  # [tokens, 2, Hkv, D]
    touched = (s["longest"] + page - 2) // page + 1  # pages of a sequence that the call may reach
    j = (start // page)[:, None] + torch.arange(touched, device=dev)  # [B, touched]
    b, i = torch.nonzero((j * page < (start + count)[:, None]) & (count > 0)[:, None], as_tuple=True)
    j, phys = j[b, i], table[b, j[b, i]].long()
    p = j[:, None] * page + torch.arange(page, device=dev)  # positions of each touched page
    t = p - start[b][:, None]
    new = ((t >= 0) & (t < count[b][:, None]))[:, None, None, :, None]
    x = rows[(first[b][:, None] + t).clamp(0, rows.shape[0] - 1)].permute(0, 2, 3, 1, 4)  # [n, 2, Hkv, page, D]
    x = torch.where(new, x, torch.zeros_like(x))
    held = pages.view(torch.uint8)[phys]
    was = torch.where((p[:, 0] < start[b])[:, None, None], scales[phys], torch.zeros_like(scales[phys]))
    scale = torch.maximum(was, _codes(x)[1])
    div = torch.where(scale > 0, scale, torch.ones_like(scale))[..., None, None]
    old = held.view(torch.float8_e4m3fn).float() * (was[..., None, None] / div)
    codes = torch.where(new, x / div, old).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = (t < count[b][:, None])[:, None, None, :, None]  # what lies past the new rows is left as it is
    pages.view(torch.uint8)[phys] = torch.where(keep, codes, held)
    scales[phys] = scale
    return {"pages": pages, "scales": scales}


def _soft(scores, seen):
    """Softmax weights of fp32 scores over the keys that are seen; a row that sees none gets zeros."""
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _attend(s):
    q, table = s["q"], s["table"].long()
    B, Hq, T, D = q.shape
    held = s["pages"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float()  # [B, P, 2, Hkv, page, D]
    held = held * s["scales"][table][..., None, None]
    Hkv, N = held.shape[3], held.shape[1] * held.shape[4]
    k, v = held.permute(2, 0, 3, 1, 4, 5).reshape(2, B, Hkv, N, D)
    key = torch.arange(N, device=q.device)
    end = s["kv_len"].long()[:, None] - T + 1 + torch.arange(T, device=q.device)  # keys that row t sees
    seen = (key < end[:, :, None])[:, None, None]
    rows = q.float().reshape(B, Hkv, Hq // Hkv, T, D)
    w = _soft(torch.matmul(rows, k[:, :, None].transpose(-1, -2)) * s["scale"], seen)
    return torch.matmul(w, v[:, :, None]).reshape(B, Hq, T, D).to(q.dtype)


def _prompts(s):
    q, k, v = s["q"][0].float(), s["k"][0].float(), s["v"][0].float()
    cu, L, dev = s["cu"].long(), s["longest"], q.device
    Hq, total, D = q.shape
    Hkv, S = k.shape[0], cu.numel() - 1
    i = torch.arange(L, device=dev)
    at = (cu[:-1, None] + i).clamp(max=total - 1)  # rows of each prompt, padded
    qp = q[:, at].reshape(Hkv, Hq // Hkv, S, L, D)
    kp, vp = k[:, at][:, None], v[:, at][:, None]
    w = _soft(torch.matmul(qp, kp.transpose(-1, -2)) * s["scale"], i[None, :] <= i[:, None])
    o = torch.matmul(w, vp).reshape(Hq, S, L, D)
    row = torch.arange(total, device=dev)
    seq = torch.bucketize(row, cu[1:], right=True)
    return o[:, seq, row - cu[seq]][None].to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------ in 64 bits


def _turned(x, position, w, layout, amp, sign):
    """One head's rows x [n, D] in fp64 rotated by the positions [n] at the angles w a position."""
    R = 2 * len(w)
    a = position.double()[:, None] * torch.tensor(w, dtype=torch.float64, device=x.device)
    z = torch.polar(torch.full_like(a, amp), sign * a)
    pair = (x[:, :R].reshape(-1, 2, R // 2).transpose(1, 2) if layout == "half" else x[:, :R].reshape(-1, R // 2, 2))
    y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
    y = y.transpose(1, 2).reshape(-1, R) if layout == "half" else y.reshape(-1, R)
    return torch.cat([y, x[:, R:]], 1)


def _nearest_code(x):
    """The e4m3 value nearest to each x (fp64, |x| <= 448), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rope":
        out = torch.empty(s["x"].shape, dtype=torch.float64, device=s["x"].device)
        w = _frequencies(c["R"], c["factor"])
        for b in range(c["B"]):
            for h in range(c["H"]):
                out[b, h] = _turned(s["x"][b, h].double(), s["positions"][b], w, c["layout"], s["amp"],
                                    -1.0 if c["inverse"] else 1.0)
        return out
    if c["op"] == "append":
        before, new = _kept(c)
        pages, scales = s["pages"].double(), s["scales"].double()
        at = 0
        for b, (n0, n) in enumerate(zip(before, new)):
            for kind, src in enumerate((s["k"], s["v"])):
                for h in range(c["Hkv"]):
                    x = (src[0, h, at:at + n] if c["packed"] else src[b, h]).double()
                    if kind == 0 and c["R"]:
                        x = _turned(x, torch.arange(n0, n0 + n, device=x.device), _frequencies(c["R"], 1.0),
                                    c["layout"], 1.0, 1.0)
                    done = 0
                    if n and n0 % c["page"]:  # the page that earlier tokens began
                        pg, lo = int(s["table"][b, n0 // c["page"]]), n0 % c["page"]
                        done = min(n, c["page"] - lo)
                        was, y = scales[pg, kind, h].item(), x[:done]
                        now = max(was, 2.0 ** math.ceil(math.log2(y.abs().max().item() / CODE_MAX)))
                        pages[pg, kind, h, :lo] = _nearest_code(pages[pg, kind, h, :lo] * (was / now))
                        pages[pg, kind, h, lo:lo + done] = _nearest_code(y / now)
                        scales[pg, kind, h] = now
                    whole = (n - done) // c["page"]
                    j0 = (n0 + done) // c["page"]
                    for y, ids in ((x[done:done + whole * c["page"]].reshape(whole, c["page"], c["D"]),
                                    s["table"][b, j0:j0 + whole].long()),
                                   (x[done + whole * c["page"]:][None], s["table"][b, j0 + whole:j0 + whole + 1].long())):
                        if y.numel():
                            now = torch.exp2(torch.ceil(torch.log2(y.abs().amax((1, 2)) / CODE_MAX)))
                            pages[ids, kind, h, :y.shape[1]] = _nearest_code(y / now[:, None, None])
                            scales[ids, kind, h] = now
            at += n
        return {"pages": pages, "scales": scales}
    G = c["Hq"] // c["Hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    if c["op"] == "attend":
        lens = _lens(c)
        for b, n in enumerate(lens):
            ids = s["table"][b, :-(-n // c["page"])].long()
            for h in range(c["Hkv"]):
                k, v = ((s["pages"].view(torch.uint8)[ids, i, h].view(torch.float8_e4m3fn).double()
                         * s["scales"][ids, i, h].double()[:, None, None]).reshape(-1, c["D"])[:n] for i in (0, 1))
                for t in range(c["T"]):
                    m = n - c["T"] + 1 + t
                    p = torch.softmax(s["q"][b, h * G:(h + 1) * G, t].double() @ k[:m].T * s["scale"], -1)
                    out[b, h * G:(h + 1) * G, t] = p @ v[:m]
        return out
    at = 0
    for n in _cuts(c["T"], c["S"]):
        hide = torch.ones(n, n, dtype=torch.bool, device=out.device).triu(1)
        for h in range(c["Hq"]):
            q, k, v = (s[x][0, y, at:at + n].double() for x, y in (("q", h), ("k", h // G), ("v", h // G)))
            out[0, h, at:at + n] = torch.softmax((q @ k.T * s["scale"]).masked_fill(hide, -math.inf), -1) @ v
        at += n
    return out
