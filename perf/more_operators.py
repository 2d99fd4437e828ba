"""Serving from a paged 8-bit KV cache that sequences share, as cases to measure: attention of chunks of new tokens over
the cached ones, copying pages (forked sequences, a pool of another size), and compacting sequences to the tokens kept.

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

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODE_MAX = 448.0  # the largest e4m3 value
BASE = 10000.0    # of the keys' rotation


def listed():
    return [
        # a short question behind a cached conversation: latency
        {"name": "chunk_question", "op": "chunk", "S": 1, "T": 33, "Hq": 32, "Hkv": 8, "D": 128, "N": 777, "page": 16,
         "dtype": "bf16"},
        # the next turns of nine conversations, uneven in new and in cached tokens
        {"name": "chunk_turns", "op": "chunk", "S": 9, "T": 1500, "Hq": 32, "Hkv": 4, "D": 128, "N": 8192, "page": 64,
         "dtype": "bf16"},
        # a slice of a long prompt that goes in piece by piece
        {"name": "chunk_long", "op": "chunk", "S": 1, "T": 2048, "Hq": 32, "Hkv": 8, "D": 128, "N": 32768, "page": 128,
         "dtype": "bf16"},
        # wide heads, many query heads a KV head, an odd number of rows
        {"name": "chunk_wide", "op": "chunk", "S": 3, "T": 1001, "Hq": 24, "Hkv": 2, "D": 256, "N": 16390, "page": 32,
         "dtype": "f16"},
        # many short turns over small pages, an odd number of query heads a KV head
        {"name": "chunk_narrow", "op": "chunk", "S": 17, "T": 4001, "Hq": 14, "Hkv": 2, "D": 64, "N": 2000, "page": 16,
         "dtype": "f16"},
        # the half-filled last pages of a few forked sequences: latency
        {"name": "copy_fork", "op": "copy", "n": 4, "Hkv": 8, "D": 128, "page": 64, "pools": 1},
        # small pages of a search with many beams
        {"name": "copy_beams", "op": "copy", "n": 333, "Hkv": 4, "D": 128, "page": 16, "pools": 1},
        # every page in use moved into a pool of another size
        {"name": "copy_pool", "op": "copy", "n": 4000, "Hkv": 8, "D": 128, "page": 64, "pools": 2},
        # one conversation cut to its first tokens and a recent window, keys turned to their new positions
        {"name": "compact_window", "op": "compact", "B": 1, "N": 4099, "kept": 1030, "way": "window", "Hkv": 8, "D": 128,
         "R": 128, "layout": "half", "page": 64},
        # a batch of sequences that each keep scattered tokens
        {"name": "compact_scattered", "op": "compact", "B": 16, "N": 8192, "kept": 4096, "way": "scattered", "Hkv": 4,
         "D": 128, "R": 128, "layout": "interleaved", "page": 32},
        # wide heads whose keys are not rotated, large pages
        {"name": "compact_wide", "op": "compact", "B": 3, "N": 16390, "kept": 11001, "way": "scattered", "Hkv": 2,
         "D": 256, "R": 0, "layout": "half", "page": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "copy", "compact"])
    D, page = rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    if op == "chunk":
        G = rng.choice([1, 3, 4, 7, 8, 12])
        S, T = _log(rng, 1, 32), _log(rng, 16, 4000)
        N = min(_log(rng, 200, 40000), 200_000 // S, 250_000_000_000 // (T * G * Hkv * D))
        return {"op": op, "S": S, "T": max(S, T), "Hq": G * Hkv, "Hkv": Hkv, "D": D, "N": max(N, 64), "page": page,
                "dtype": rng.choice(["bf16", "f16"])}
    if op == "copy":
        n = min(_log(rng, 1, 6000), max(1, 500_000_000 // (2 * Hkv * D * page)))
        return {"op": op, "n": n, "Hkv": Hkv, "D": D, "page": page, "pools": rng.choice([1, 2])}
    B = _log(rng, 1, 24)
    N = min(_log(rng, 150, 30000), 300_000_000 // (B * 2 * Hkv * D))
    return {"op": op, "B": B, "N": N, "kept": max(1, int(N * rng.uniform(0.1, 0.9))),
            "way": rng.choice(["window", "scattered"]), "Hkv": Hkv, "D": D, "R": rng.choice([0, D // 2, D]),
            "layout": rng.choice(["half", "interleaved"]), "page": page}


# ------------------------------------------------------------------------------------------------ lengths of a case


def _cuts(total, parts):
    """`parts` uneven lengths, all above 0, that sum to `total`."""
    rng = random.Random(total * 1013 + parts)
    w = [rng.random() ** 2 + 0.02 for _ in range(parts)]
    at = [int((total - parts) * sum(w[:i]) / sum(w)) for i in range(parts)] + [total - parts]
    return [at[i + 1] - at[i] + 1 for i in range(parts)]


def _lens(c):
    """New tokens of each sequence, and its cached ones with them."""
    rng = random.Random(c["S"] * 7927 + c["N"])
    new = _cuts(c["T"], c["S"])
    return new, [max(n, c["N"] if i == 0 else rng.randint(c["N"] // 2, c["N"])) for i, n in enumerate(new)]


def _sizes(c):
    """Tokens of each sequence of a compaction, and how many of them are kept."""
    rng = random.Random(c["B"] * 7933 + c["N"])
    have = [c["N"] if i == 0 else rng.randint(max(1, c["N"] // 2), c["N"]) for i in range(c["B"])]
    return have, [max(1, min(n, n * c["kept"] // c["N"])) for n in have]


def work(c):
    if c["op"] == "chunk":
        new, lens = _lens(c)
        pairs = sum(n * (2 * m - n + 1) // 2 for n, m in zip(new, lens))
        return {"bytes": 2.0 * sum(lens) * c["Hkv"] * c["D"] + 4.0 * c["T"] * c["Hq"] * c["D"],
                "flops": 4.0 * pairs * c["Hq"] * c["D"]}
    if c["op"] == "copy":
        return {"bytes": 2.0 * c["n"] * 2 * c["Hkv"] * (c["page"] * c["D"] + 4), "flops": 0.0}
    kept = sum(_sizes(c)[1])
    return {"bytes": 2.0 * kept * 2 * c["Hkv"] * c["D"], "flops": 3.0 * kept * c["Hkv"] * c["R"]}


# ------------------------------------------------------------------------------------------------ inputs


def _angles(R):
    """Angles a position, in radians."""
    return [BASE ** (-2 * i / R) for i in range(R // 2)]


def _turns(R, dev):
    """The same as 64-bit fractions of a turn, which a position multiplies exactly."""
    f = [int(round(w / (2 * math.pi) * 2.0 ** 64)) for w in _angles(R)]
    return torch.tensor([x - (1 << 64) if x >= 1 << 63 else x for x in f], dtype=torch.int64, device=dev)


def _codes(x):
    """Pages x [..., page, D] fp32 as e4m3 codes and their power-of-two scales [...]."""
    m = x.abs().amax((-2, -1))
    f, e = torch.frexp(m)  # m = f 2^e, f in [1/2, 1): exact, as a page's largest value may well be 448 s itself
    s = torch.where(m > 0, torch.ldexp(torch.ones_like(m), e - 9 + (f > CODE_MAX / 512)), torch.zeros_like(m))
    return torch.where(s[..., None, None] > 0, x / s[..., None, None], torch.zeros_like(x)).to(torch.float8_e4m3fn), s


def _pool(gen, dev, num, page, Hkv, D):
    """A pool of filled pages whose loudness differs from page to page."""
    pages = torch.empty(num, 2, Hkv, page, D, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(num, 2, Hkv, device=dev)
    loud = torch.ones(2, 1, 1, D, device=dev)
    loud[0, :, :, ::37] = 6.0  # a few loud key channels
    step = max(1, (1 << 26) // (2 * Hkv * page * D))
    for i in range(0, num, step):
        n = min(step, num - i)
        x = torch.randn(n, 2, Hkv, page, D, generator=gen, device=dev) * loud
        x *= torch.exp(0.3 * torch.randn(n, 2, Hkv, 1, 1, generator=gen, device=dev))
        p, scales[i:i + step] = _codes(x)
        pages.view(torch.uint8)[i:i + step] = p.view(torch.uint8)
    return pages, scales


def _table(order, per, dev):
    """Page tables of sequences of per[b] pages, taken from `order` in turn."""
    table = torch.zeros(len(per), max(per), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    page, Hkv, D = c["page"], c["Hkv"], c["D"]
    s = {"op": c["op"]}
    if c["op"] == "copy":
        num = c["n"] * (2 if c["pools"] == 1 else 1) + 3
        s["pages"], s["scales"] = _pool(gen, dev, num, page, Hkv, D)
        order = torch.randperm(num, generator=gen, device=dev).to(torch.int32)
        s["src"] = order[:c["n"]].contiguous()
        s["into"] = None
        if c["pools"] == 1:
            s["dst"] = order[c["n"]:2 * c["n"]].contiguous()
        else:
            s["into"] = (torch.zeros_like(s["pages"].view(torch.uint8)).view(torch.float8_e4m3fn),
                         torch.zeros_like(s["scales"]))
            s["dst"] = torch.arange(c["n"], dtype=torch.int32, device=dev)
        return s
    if c["op"] == "chunk":
        new, lens = _lens(c)
        per = [-(-n // page) for n in lens]
        num = sum(per) + 3
        s["pages"], s["scales"] = _pool(gen, dev, num, page, Hkv, D)
        s["table"] = _table(torch.randperm(num, generator=gen, device=dev).to(torch.int32), per, dev)
        s["new"], s["lens"] = new, lens  # what the program that admits the tokens knows
        s["kv_len"], s["cu"] = _ints(lens, dev), _ints(_starts(new), dev)
        rows = torch.randn(1, c["T"], c["Hq"], D, generator=gen, device=dev)  # token-major, as a projection leaves them
        s["q"] = rows.to(DTYPES[c["dtype"]]).transpose(1, 2)
        s["scale"] = D ** -0.5
        return s
    have, kept = _sizes(c)
    keep, start, flat = [], [], []
    host = random.Random(seed)
    for n, m in zip(have, kept):
        if c["way"] == "window":
            first = min(4, m)
            at = list(range(first)) + list(range(n - (m - first), n))
        else:
            at = sorted(host.sample(range(n), m))
        same = 0
        while same < m and at[same] == same:
            same += 1
        same = same // page * page  # whole pages that stay as they are
        start.append(same)
        keep.append(at[same:])
        flat += at[same:]
    per, to = [-(-n // page) for n in have], [-(-m // page) for m in kept]
    num = sum(per) + sum(to) + 3
    s["pages"], s["scales"] = _pool(gen, dev, num, page, Hkv, D)
    order = torch.randperm(num, generator=gen, device=dev).to(torch.int32)
    s["table"], s["to"] = _table(order, per, dev), _table(order[sum(per):], to, dev)
    s["keep"], s["cu"], s["start"] = _ints(flat, dev), _ints(_starts([len(k) for k in keep]), dev), _ints(start, dev)
    s["longest"] = max(len(k) for k in keep)
    s["turns"], s["layout"] = (_turns(c["R"], dev) if c["R"] else None), c["layout"]
    return s


# ------------------------------------------------------------------------------------------------ the operators


def run(s):
    if own:
        from larder_b200 import ops
        if s["op"] == "chunk":
            return ops.kv8_attend_packed(s["q"], s["pages"], s["scales"], s["table"], s["kv_len"], s["cu"], s["scale"])
        if s["op"] == "copy":
            ops.kv8_copy(s["pages"], s["scales"], s["src"], s["dst"], into=s["into"])
            return s["into"] or (s["pages"], s["scales"])
        ops.kv8_compact(s["pages"], s["scales"], s["table"], s["keep"], s["cu"], s["to"], s["start"], turns=s["turns"],
                        layout=s["layout"])
        return s["pages"], s["scales"]
    return {"chunk": _chunk, "copy": _copy, "compact": _compact}[s["op"]](s)


def _chunk(s):
    q, page = s["q"][0], s["pages"].shape[3]
    Hq, total, D = q.shape
    Hkv = s["pages"].shape[2]
    out = torch.zeros(1, Hq, total, D, dtype=q.dtype, device=q.device)
    at = 0
    for b, (n, m) in enumerate(zip(s["new"], s["lens"])):
        ids = s["table"][b, :-(-m // page)].long()
        held = s["pages"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * s["scales"][ids][..., None, None]
        k, v = held.permute(1, 2, 0, 3, 4).reshape(2, Hkv, 1, -1, D)[:, :, :, :m]
        key = torch.arange(m, device=q.device)
        step = max(1, (1 << 28) // (Hq * m))  # rows whose scores stay within a gigabyte
        for i in range(0, n, step):
            j = min(n, i + step)
            rows = q[:, at + i:at + j].float().reshape(Hkv, Hq // Hkv, j - i, D)
            sc = torch.matmul(rows, k.transpose(-1, -2)) * s["scale"]
            seen = key <= (m - n + torch.arange(i, j, device=q.device))[:, None]
            sc = torch.where(seen, sc, torch.full_like(sc, -math.inf))
            e = torch.exp(sc - sc.amax(-1, keepdim=True))  # (a row sees itself at least)
            o = torch.matmul(e / e.sum(-1, keepdim=True), v)
            out[0, :, at + i:at + j] = o.reshape(Hq, j - i, D).to(q.dtype)
        at += n
    return out


def _copy(s):
    pages, scales = s["into"] or (s["pages"], s["scales"])
    src, dst = s["src"].long(), s["dst"].long()
    pages.view(torch.uint8)[dst] = s["pages"].view(torch.uint8)[src]
    scales[dst] = s["scales"][src]
    return pages, scales


def _rotate(x, positions, turns, layout):
    """x [n, Hkv, D] fp32 with its first 2 len(turns) dims rotated by the positions [n] (of either sign)."""
    R = 2 * turns.numel()
    a = (positions[:, None, None] * turns).float() * (2 * math.pi / 2.0 ** 64)
    c, n = torch.cos(a), torch.sin(a)
    if layout == "half":
        x0, x1 = x[..., :R // 2], x[..., R // 2:R]
        y = torch.cat([x0 * c - x1 * n, x1 * c + x0 * n], -1)
    else:
        x0, x1 = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack([x0 * c - x1 * n, x1 * c + x0 * n], -1).flatten(-2)
    return torch.cat([y, x[..., R:]], -1)


def _compact(s):
    pages, scales, table, to = s["pages"], s["scales"], s["table"].long(), s["to"].long()
    _, _, Hkv, page, D = pages.shape
    raw, dev = pages.view(torch.uint8), pages.device
    cu, start, keep = s["cu"].long(), s["start"].long(), s["keep"].long()
    count = cu[1:] - cu[:-1]
    row = torch.arange(keep.numel(), device=dev)
    seq = torch.bucketize(row, cu[1:], right=True)
    ids = table[seq, keep // page]
    x = raw[ids, :, :, keep % page].view(torch.float8_e4m3fn).float() * scales[ids][..., None]  # [tokens, 2, Hkv, D]
    if s["turns"] is not None:
        x[:, 0] = _rotate(x[:, 0], row - cu[seq] + start[seq] - keep, s["turns"], s["layout"])
    j = torch.arange(-(-s["longest"] // page), device=dev)
    b, i = torch.nonzero(j * page < count[:, None], as_tuple=True)
    phys = to[b, start[b] // page + i]
    t = i[:, None] * page + torch.arange(page, device=dev)  # [pages, page] of the sequence's moved tokens
    new = (t < count[b][:, None])[:, None, None, :, None]
    y = x[(cu[b][:, None] + t).clamp(max=keep.numel() - 1)].permute(0, 2, 3, 1, 4)
    codes, scale = _codes(torch.where(new, y, torch.zeros_like(y)))
    raw[phys] = torch.where(new, codes.view(torch.uint8), raw[phys])  # what lies past the last token stays
    scales[phys] = scale
    return pages, scales


# ------------------------------------------------------------------------------------------------ in 64 bits


def _nearest_code(x):
    """The e4m3 value nearest to each x (fp64, |x| <= 448), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(c, seed):
    s = prepare(c, seed)
    page = c["page"]
    if c["op"] == "copy":
        pages, scales = (t.double() for t in (s["into"] or (s["pages"], s["scales"])))
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pages[b], scales[b] = s["pages"][a].double(), s["scales"][a].double()
        return pages, scales

    def rows(b, kind, h, at):
        """Held values of a sequence's positions `at`, fp64 [n, D]."""
        ids = s["table"][b, at // page].long()
        codes = s["pages"].view(torch.uint8)[ids, kind, h, at % page].view(torch.float8_e4m3fn).double()
        return codes * s["scales"][ids, kind, h].double()[:, None]

    if c["op"] == "chunk":
        q = s["q"]
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        G, at = c["Hq"] // c["Hkv"], 0
        for b, (n, m) in enumerate(zip(*_lens(c))):
            hide = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
            everything = torch.arange(m, device=q.device)
            for hk in range(c["Hkv"]):
                k, v = rows(b, 0, hk, everything), rows(b, 1, hk, everything)
                for h in range(hk * G, hk * G + G):
                    sc = (q[0, h, at:at + n].double() @ k.T * s["scale"]).masked_fill_(hide, -math.inf)
                    out[0, h, at:at + n] = torch.softmax(sc, -1) @ v
            at += n
        return out
    pages, scales = s["pages"].double(), s["scales"].double()
    cu, start = s["cu"].tolist(), s["start"].tolist()
    w = torch.tensor(_angles(c["R"]), dtype=torch.float64, device=pages.device) if c["R"] else None
    for b in range(c["B"]):
        at = s["keep"][cu[b]:cu[b + 1]].long()
        n = at.numel()
        if n == 0:
            continue
        turn = None
        if c["R"]:
            a = (torch.arange(n, device=at.device) + start[b] - at).double()[:, None] * w
            turn = torch.polar(torch.ones_like(a), a)
        ids = s["to"][b, start[b] // page:].long()[:-(-n // page)]
        for kind in (0, 1):
            for h in range(c["Hkv"]):
                x = rows(b, kind, h, at)
                if kind == 0 and c["R"]:
                    R, z = c["R"], x[:, :c["R"]]
                    pair = z.reshape(n, 2, R // 2).transpose(1, 2) if c["layout"] == "half" else z.reshape(n, R // 2, 2)
                    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
                    z = z.transpose(1, 2).reshape(n, R) if c["layout"] == "half" else z.reshape(n, R)
                    x = torch.cat([z, x[:, R:]], 1)
                whole = n // page
                for y, to in ((x[:whole * page].reshape(whole, page, -1), ids[:whole]),
                              (x[whole * page:][None], ids[whole:])):
                    if y.numel():
                        top = y.abs().amax((1, 2))
                        now = torch.exp2(torch.floor(torch.log2(top)) - 9)
                        for _ in range(2):
                            now = torch.where(top > CODE_MAX * now, 2 * now, now)
                        pages[to, kind, h, :y.shape[1]] = _nearest_code(y / now[:, None, None])
                        scales[to, kind, h] = now
    return pages, scales
