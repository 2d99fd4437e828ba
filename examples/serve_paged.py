"""Serving with the paged 8-bit KV cache: prompts admitted together, decoded together, one of them ended and replaced.

    python examples/serve_paged.py [--steps N]

One attention layer with random weights stands for the model: q, k, v projections of a hidden state, rotary positions,
attention, the output projection, whose result is the next step's hidden state. Prompts go in packed on one row axis
(attn_packed over the prompt's own keys, then the keys and values into the cache); each decode step appends one token a
sequence and attends over the cache. Prints the steps' time and how far the cached attention is from attention over the
unrounded keys and values.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from larder_b200 import kv8, ops  # noqa: E402
from larder_b200.rope import Rope  # noqa: E402


class Layer:
    def __init__(self, hidden, hq, hk, d, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.hq, self.hk, self.d = hq, hk, d
        self.qkv = torch.randn(hidden, (hq + 2 * hk) * d, generator=g, device=device).mul_(hidden ** -0.5).to(torch.bfloat16)
        self.out = torch.randn(hq * d, hidden, generator=g, device=device).mul_((hq * d) ** -0.5).to(torch.bfloat16)
        self.rope = Rope(d, base=1e6, scaling={"kind": "yarn", "factor": 4.0, "original": 32768}, device=device)
        self.scale = d ** -0.5

    def project(self, x):
        """x [B, T, hidden] -> q [B, hq, T, d], k, v [B, hk, T, d], views of one projection's rows."""
        rows = (x @ self.qkv).unflatten(-1, (-1, self.d)).transpose(1, 2)
        return rows.split([self.hq, self.hk, self.hk], 1)

    def finish(self, o):
        return o.transpose(1, 2).flatten(2) @ self.out

    def prompts(self, cache, handles, x, lens):
        """Hidden states x [1, sum(lens), hidden] of new sequences' prompts, packed; their last rows' outputs."""
        step = cache.step(handles, lens)
        q, k, v = self.project(x)
        pos = step.positions.reshape(-1)
        o = ops.attn_packed(self.rope.apply(q, pos), self.rope.apply(k, pos), v, self.scale, step.cu)
        cache.append(step, k, v, rope=self.rope, packed=True)
        return self.finish(o)[0, step.cu[1:].long() - 1][:, None]

    def decode(self, cache, handles, x):
        """One token of each sequence: hidden states x [B, 1, hidden]."""
        step = cache.step(handles, [1] * len(handles))
        q, k, v = self.project(x)
        cache.append(step, k, v, rope=self.rope)
        return self.finish(cache.attend(step, self.rope.apply(q, step.positions), self.scale)), (step, q, k, v)


def main(steps=32, hidden=2048, hq=32, hk=8, d=128, lens=(700, 1500, 33, 260), device="cuda"):
    layer = Layer(hidden, hq, hk, d, device)
    cache = kv8.Cache(num_pages=512, page=64, hk=hk, d=d, device=device)
    g = torch.Generator(device=device).manual_seed(1)

    def prompt(n):
        return torch.randn(1, n, hidden, generator=g, device=device).to(torch.bfloat16)

    handles = [cache.add() for _ in lens]
    first = prompt(sum(lens))
    x = layer.prompts(cache, handles, first, list(lens))
    kept = [tuple(t[:, :, a:a + n] for t in layer.project(first)[1:]) for a, n in zip([sum(lens[:i]) for i in range(len(lens))], lens)]
    worst, start, end = 0.0, torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(steps):
        y, (step, q, k, v) = layer.decode(cache, handles, x)
        kept = [(torch.cat([a, k[i:i + 1]], 2), torch.cat([b, v[i:i + 1]], 2)) for i, (a, b) in enumerate(kept)]
        x = y
    end.record()
    torch.cuda.synchronize()
    # the last step again, over the unrounded keys and values
    q = layer.rope.apply(q, step.positions)
    o = cache.attend(step, q, layer.scale).float()
    for i, (a, b) in enumerate(kept):
        ka = layer.rope.apply(a.contiguous(), torch.arange(a.shape[2], dtype=torch.int32, device=device)).float()
        ka, va = (t[0].float().repeat_interleave(hq // hk, 0) for t in (ka, b))
        ref = torch.softmax(torch.einsum("hd,hnd->hn", q[i, :, 0].float(), ka) * layer.scale, -1)
        ref = torch.einsum("hn,hnd->hd", ref, va)
        worst = max(worst, ((o[i, :, 0] - ref).norm() / ref.norm()).item())
    print(f"{steps} decode steps of {len(lens)} sequences: {start.elapsed_time(end) / steps * 1e3:.0f} us a step "
          f"(with this script's own copies); 8-bit cache against unrounded keys and values: {worst:.3f} relative")
    # one sequence ends, another takes its pages
    cache.drop(handles.pop(1))
    new = cache.add()
    x = torch.cat([x[[0, 2, 3]], layer.prompts(cache, [new], prompt(90), [90])])
    handles.append(new)
    for _ in range(3):
        x, _ = layer.decode(cache, handles, x)
    assert ops.status() == 0 and torch.isfinite(x).all()
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=32)
    main(steps=ap.parse_args().steps)
