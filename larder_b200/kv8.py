"""A paged KV cache in 8 bits: e4m3 codes with a power-of-two scale for each page and head of K and of V.

    cache = Cache(num_pages=4096, page=64, hk=8, d=128)
    a, b = cache.add(), cache.add()                   # two sequences
    step = cache.step([a, b], [700, 12])              # room for their prompts: page table, first positions, lengths
    cache.append(step, k, v, rope=rope, packed=True)  # k / v [1, hk, 712, d], keys rotated on the way
    step = cache.step([a, b], [1, 1])                 # one decode step
    cache.append(step, k1, v1, rope=rope)             # [2, hk, 1, d]
    o = cache.attend(step, q1, scale)                 # q1 [2, hq, 1, d], rotated by rope.apply(q1, step.positions)
    cache.drop(b)                                     # its pages are free again

Pages are handed out on the host; the device sees a page table a step. The codes, the rounding and what the kernels
check are lb2_kv8_append's and lb2_kv8_attend's.
"""
import torch

from . import ops


class Step:
    """One call's sequences: table int32 [B, max_pages], start and kv_len int32 [B] (tokens before and after the call),
    cu int32 [B + 1] (row offsets of the new tokens packed), positions int32 (of the new tokens: [B, T] where every
    sequence has T, else packed [rows])."""

    def __init__(self, table, start, kv_len, cu, positions, counts, spans=()):
        self.table, self.start, self.kv_len, self.cu = table, start, kv_len, cu
        self.positions, self.counts = positions, counts
        self.spans = spans  # (handle, tokens before the call, new tokens) of each sequence, on the host


class Cache:
    def __init__(self, num_pages, page, hk, d, device="cuda"):
        if page not in (16, 32, 64, 128) or d not in (64, 128, 256) or num_pages < 1 or hk < 1:
            raise ValueError("kv8: pages of 16, 32, 64 or 128 tokens, head dim 64, 128 or 256, at least one page and head")
        self.page, self.hk, self.d = page, hk, d
        self.device = torch.device(device)
        self.pages = torch.zeros((num_pages, 2, hk, page, d), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.scales = torch.zeros((num_pages, 2, hk), dtype=torch.float32, device=device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._seqs = {}  # handle -> [page ids, tokens]
        self._missing = {}  # handle -> first positions of the steps whose append was refused
        self._next = 0

    @property
    def free_pages(self):
        return len(self._free)

    def add(self):
        """A new, empty sequence's handle."""
        h = self._next
        self._next += 1
        self._seqs[h] = [[], 0]
        return h

    def drop(self, handle):
        """Ends a sequence; its pages may be handed out again."""
        self._free.extend(reversed(self._seqs.pop(handle)[0]))
        self._missing.pop(handle, None)

    def length(self, handle):
        return self._seqs[handle][1]

    def trim(self, handle, n):
        """Forgets a sequence's tokens from position n on (rejected drafts). The kept page's scale stays as it is."""
        ids, have = self._seqs[handle]
        if not 0 <= n <= have:
            raise ValueError(f"kv8: cannot trim a sequence of {have} tokens to {n}")
        keep = -(-n // self.page)
        self._free.extend(reversed(ids[keep:]))
        del ids[keep:]
        self._seqs[handle][1] = n
        for s in [s for s in self._missing.get(handle, ()) if s >= n]:
            self._found(handle, s)

    def _found(self, handle, start):
        starts = self._missing.get(handle, set())
        starts.discard(start)
        if not starts:
            self._missing.pop(handle, None)

    def step(self, handles, counts):
        """Reserves room for counts[i] new tokens of handles[i] and returns the call's Step. Nothing is reserved, and a
        ValueError raised, when the pool has too few free pages."""
        if len(set(handles)) != len(handles) or len(handles) != len(counts) or any(c < 0 for c in counts):
            raise ValueError("kv8: distinct sequences, one count each")
        need = [max(0, -(-(self._seqs[h][1] + c) // self.page) - len(self._seqs[h][0])) for h, c in zip(handles, counts)]
        if sum(need) > len(self._free):
            raise ValueError(f"kv8: {sum(need)} pages needed, {len(self._free)} free")
        start = []
        for h, c, n in zip(handles, counts, need):
            seq = self._seqs[h]
            seq[0].extend(self._free.pop() for _ in range(n))
            start.append(seq[1])
            seq[1] += c
        width = max([1] + [len(self._seqs[h][0]) for h in handles])
        rows = [self._seqs[h][0] + [0] * (width - len(self._seqs[h][0])) for h in handles]
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        positions = [s + i for s, c in zip(start, counts) for i in range(c)]
        B = len(handles)
        # one copy to the device: the table, start, kv_len, cu and positions in turn
        flat = [x for r in rows for x in r] + start + [s + c for s, c in zip(start, counts)] + cu + positions
        t = torch.tensor(flat, dtype=torch.int32).to(self.device)
        table, start_t, len_t, cu_t, pos = t.split([B * width, B, B, B + 1, len(positions)])
        same = B and all(c == counts[0] for c in counts)
        return Step(table.view(B, width), start_t, len_t, cu_t, pos.view(B, counts[0]) if same else pos, list(counts),
                    list(zip(handles, start, counts)))

    def append(self, step, k, v, rope=None, packed=False):
        """The step's new tokens: k / v [B, hk, T, d] where every sequence has T of them, or, packed, [1, hk, rows, d].
        Keys are rotated by their positions when a Rope is given. After a refused append the step's tokens still count:
        append them again, or trim them away; attend refuses sequences that lack them."""
        try:
            kw = {} if rope is None else {"turns": rope.turns, "layout": rope.layout, "amp": rope.amp}
            if packed:
                if k.shape[2] != sum(step.counts):
                    raise ValueError(f"kv8: {sum(step.counts)} packed rows expected, got {k.shape[2]}")
                kw["cu"] = step.cu
            elif any(c != k.shape[2] for c in step.counts):
                raise ValueError("kv8: sequences with different counts go in packed")
            ops.kv8_append(self.pages, self.scales, k, v, step.table, step.start, **kw)
        except Exception:  # the step's tokens count, but the pages do not hold them
            for h, s, n in step.spans:
                if n and h in self._seqs:
                    self._missing.setdefault(h, set()).add(s)
            raise
        if self._missing:
            for h, s, n in step.spans:
                if n:
                    self._found(h, s)

    def attend(self, step, q, scale, causal=True, out=None):
        """q [B, hq, T, d], the queries of each sequence's last T tokens, over everything cached."""
        if self._missing:
            for h, s, n in step.spans:
                if any(x < s + n for x in self._missing.get(h, ())):
                    raise ValueError(f"kv8: sequence {h} has tokens that were not appended (their append was refused)")
        return ops.kv8_attend(q, self.pages, self.scales, step.table, step.kv_len, scale, causal, out)


__all__ = ["Cache", "Step"]
