"""A paged KV cache in 8 bits: e4m3 codes with a power-of-two scale for each page and head of K and of V.

    cache = Cache(num_pages=4096, page=64, hk=8, d=128)
    a, b = cache.add(), cache.add()                   # two sequences
    step = cache.step([a, b], [700, 12])              # room for their prompts: page table, first positions, lengths
    cache.append(step, k, v, rope=rope, packed=True)  # k / v [1, hk, 712, d], keys rotated on the way
    step = cache.step([a, b], [1, 1])                 # one decode step
    cache.append(step, k1, v1, rope=rope)             # [2, hk, 1, d]
    o = cache.attend(step, q1, scale)                 # q1 [2, hq, 1, d], rotated by rope.apply(q1, step.positions)
    c = cache.fork(a)                                 # a sequence that begins with a's tokens, sharing their pages
    step = cache.step([b, c], [3, 40])                # the next turns, uneven
    cache.append(step, k2, v2, rope=rope, packed=True)
    o = cache.attend(step, q2, scale, packed=True)    # q2 [1, hq, 43, d]
    cache.keep([a], [list(range(4)) + list(range(400, 701))], rope)  # forget the others, keys turned to their new places
    cache.drop(b)                                     # its pages are free again
    cache.resize(1024)                                # the pages in use in a smaller pool

Pages are handed out on the host; the device sees a page table a step. A page may belong to several sequences that began
alike: it is copied for the one that appends into it. The codes, the rounding and what the kernels check are
lb2_kv8_append's, lb2_kv8_attend's, lb2_kv8_attend_packed's, lb2_kv8_copy's and lb2_kv8_compact's.
"""
import weakref

import torch

from . import ops


class _Use:
    """What a step relies on: each sequence's tokens up to the end of its span; why[handle]: what has happened to them since."""
    __slots__ = ("spans", "ends", "why", "__weakref__")

    def __init__(self, spans):
        self.spans, self.ends, self.why = spans, None, {}

    def overtake(self, handle, n, why):
        if self.ends is None:
            self.ends = {h: s + c for h, s, c in self.spans}
        if self.ends.get(handle, 0) > n:
            self.why.setdefault(handle, why)


class Step:
    """One call's sequences: table int32 [B, max_pages], start and kv_len int32 [B] (tokens before and after the call),
    cu int32 [B + 1] (row offsets of the new tokens packed), positions int32 (of the new tokens: [B, T] where every
    sequence has T, else packed [rows])."""

    def __init__(self, table, start, kv_len, cu, positions, counts, spans=(), use=None):
        self.table, self.start, self.kv_len, self.cu = table, start, kv_len, cu
        self.positions, self.counts = positions, counts
        self.spans = spans  # (handle, tokens before the call, new tokens) of each sequence, on the host
        self.use = _Use(spans) if use is None else use


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
        self._refs = [0] * num_pages  # sequences that hold each page
        self._missing = {}  # handle -> first positions of the steps whose append was refused
        self._pending = {}  # handle -> first positions of the steps whose append has not been made
        self._uses = weakref.WeakSet()  # of the steps that are still held
        self._forked = False  # some pages may be shared
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
        """Ends a sequence; its pages may be handed out again where no other sequence holds them."""
        self._release(reversed(self._seqs.pop(handle)[0]))
        for d in (self._missing, self._pending):
            d.pop(handle, None)
        self._overtake(handle, 0, f"sequence {handle} was dropped")

    def _take(self):
        i = self._free.pop()
        self._refs[i] = 1
        return i

    def _release(self, ids):
        for i in ids:
            self._refs[i] -= 1
            if not self._refs[i]:
                self._free.append(i)

    def _overtake(self, handle, n, why):
        """A sequence's tokens from position n on are no longer where steps made before have them."""
        for use in list(self._uses):
            use.overtake(handle, n, why)

    def _moved(self, handle, n):
        self._overtake(handle, n, f"sequence {handle}'s pages have moved")

    def _current(self, step, new=False):
        """Refuses a step whose tokens (new: its new ones) are no longer where it has them."""
        for h, _, n in step.spans if step.use.why else ():
            if h in step.use.why and (n or not new):
                raise ValueError(f"kv8: {step.use.why[h]} since this step was made")

    def _settled(self, handle, n=None):
        """Refuses a sequence among whose first n tokens (all) some were reserved by a step and not appended, or were to be
        appended again and that was refused."""
        if any(n is None or s < n for d in (self._pending, self._missing) for s in d.get(handle, ())):
            raise ValueError(f"kv8: sequence {handle} has tokens that a step reserved and that were not appended")

    def _lacks(self, step, where=lambda h, s: True):
        """The step's append was refused: its tokens count, but the pages do not hold them."""
        for h, s, n in step.spans:
            if n and h in self._seqs and where(h, s):
                self._missing.setdefault(h, set()).add(s)

    def length(self, handle):
        return self._seqs[handle][1]

    def trim(self, handle, n):
        """Forgets a sequence's tokens from position n on (rejected drafts). The kept page's scale stays as it is. Steps that
        reach past n are refused from now on."""
        ids, have = self._seqs[handle]
        if not 0 <= n <= have:
            raise ValueError(f"kv8: cannot trim a sequence of {have} tokens to {n}")
        keep = -(-n // self.page)
        self._release(reversed(ids[keep:]))
        del ids[keep:]
        self._seqs[handle][1] = n
        self._overtake(handle, n, f"sequence {handle} was cut to {n} tokens")
        for d in (self._missing, self._pending):
            for s in [s for s in d.get(handle, ()) if s >= n]:
                self._found(d, handle, s)

    @staticmethod
    def _found(starts_of, handle, start):
        starts = starts_of.get(handle, set())
        starts.discard(start)
        if not starts:
            starts_of.pop(handle, None)

    def fork(self, handle, n=None):
        """A new sequence that begins with another's first n tokens (all of them), sharing their pages; a page is copied
        when one of the sequences that hold it appends into it. The tokens must have been appended."""
        ids, have = self._seqs[handle]
        n = have if n is None else n
        if not 0 <= n <= have:
            raise ValueError(f"kv8: cannot fork {n} tokens of a sequence of {have}")
        self._settled(handle, n)
        shared = ids[:-(-n // self.page)]
        new = self.add()
        self._forked = True
        self._seqs[new] = [list(shared), n]
        for i in shared:
            self._refs[i] += 1
        return new

    def keep(self, handles, positions, rope=None):
        """Forgets all tokens of each sequence but those at positions[i] (rising), which become its first ones, in new
        pages where they move; codes are rounded again at the new pages' scales. With the Rope that the keys were appended
        with, keys are turned to their new positions; without one they stay as they were rotated. Refused, and nothing done,
        when the pool has too few free pages (the pages moved from are free only afterwards)."""
        if len(set(handles)) != len(handles) or len(handles) != len(positions):
            raise ValueError("kv8: distinct sequences, a list of positions each")
        positions = [list(at) for at in positions]
        moves, need = [], 0
        for h, at in zip(handles, positions):
            have = self._seqs[h][1]
            if at and not (at[0] >= 0 and at[-1] < have and all(x < y for x, y in zip(at, at[1:]))):
                raise ValueError(f"kv8: positions to keep must rise within 0 .. {have - 1}")
            self._settled(h)
            same = 0
            while same < len(at) and at[same] == same:
                same += 1
            if same < len(at):
                same -= same % self.page  # whole pages that stay
                moves.append((h, at, same))
                need += -(-(len(at) - same) // self.page)
        if need > len(self._free):
            raise ValueError(f"kv8: {need} pages needed, {len(self._free)} free")
        kw = {} if rope is None else {"turns": rope.turns, "layout": rope.layout}
        if moves:
            old = [self._seqs[h][0] for h, _, _ in moves]
            new = [ids[:same // self.page] + [self._take() for _ in range(-(-(len(at) - same) // self.page))]
                   for ids, (_, at, same) in zip(old, moves)]
            try:
                wide, wide_new = max(map(len, old)), max(map(len, new))
                cu = [0]
                for _, at, same in moves:
                    cu.append(cu[-1] + len(at) - same)
                B = len(moves)
                flat = ([x for r in old for x in r + [0] * (wide - len(r))]
                        + [x for r in new for x in r + [0] * (wide_new - len(r))]
                        + [same for _, _, same in moves] + cu + [x for _, at, same in moves for x in at[same:]])
                t = torch.tensor(flat, dtype=torch.int32).to(self.device)
                table, to, start, cu_t, keep = t.split([B * wide, B * wide_new, B, B + 1, cu[-1]])
                ops.kv8_compact(self.pages, self.scales, table.view(B, wide), keep, cu_t, to.view(B, wide_new), start, **kw)
            except Exception:
                for ids, (_, _, same) in zip(new, moves):
                    self._release(reversed(ids[same // self.page:]))
                raise
            for ids, now, (h, at, same) in zip(old, new, moves):
                self._release(reversed(ids[same // self.page:]))
                self._seqs[h] = [now, len(at)]
                self._moved(h, same)
        moved = {h for h, _, _ in moves}
        for h, at in zip(handles, positions):
            if h not in moved:
                self.trim(h, len(at))

    def resize(self, num_pages):
        """Moves the pages in use into a pool of num_pages and lets the old one go: pages and scales are new tensors, steps
        made before are refused. Every reserved token must have been appended."""
        used = [i for i, r in enumerate(self._refs) if r]
        if num_pages < 1 or len(used) > num_pages:
            raise ValueError(f"kv8: {len(used)} pages are in use, they do not fit a pool of {num_pages}")
        for h in self._seqs:
            self._settled(h)
        pages = torch.zeros((num_pages,) + self.pages.shape[1:], dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn)
        scales = torch.zeros((num_pages,) + self.scales.shape[1:], dtype=torch.float32, device=self.device)
        if used:
            t = torch.tensor(used + list(range(len(used))), dtype=torch.int32).to(self.device)
            ops.kv8_copy(self.pages, self.scales, *t.split(len(used)), into=(pages, scales))
        at = {i: j for j, i in enumerate(used)}
        for seq in self._seqs.values():
            seq[0] = [at[i] for i in seq[0]]
        self._refs = [self._refs[i] for i in used] + [0] * (num_pages - len(used))
        self._free = list(range(num_pages - 1, len(used) - 1, -1))
        self.pages, self.scales = pages, scales
        for h in self._seqs:
            self._moved(h, -1)

    def step(self, handles, counts):
        """Reserves room for counts[i] new tokens of handles[i] and returns the call's Step. Nothing is reserved, and a
        ValueError raised, when the pool has too few free pages."""
        if len(set(handles)) != len(handles) or len(handles) != len(counts) or any(c < 0 for c in counts):
            raise ValueError("kv8: distinct sequences, one count each")
        need, copies, left = [], [], {}
        for h, c in zip(handles, counts):
            ids, have = self._seqs[h]
            need.append(max(0, -(-(have + c) // self.page) - len(ids)))
            if c and have % self.page and self._refs[ids[have // self.page]] > 1:
                i = ids[have // self.page]  # the new tokens begin in a page that others hold too: the last of them keeps it
                left[i] = left.get(i, self._refs[i]) - 1
                if left[i]:
                    copies.append((h, have // self.page, i))
        if sum(need) + len(copies) > len(self._free):
            raise ValueError(f"kv8: {sum(need) + len(copies)} pages needed, {len(self._free)} free")
        dst = []
        for h, j, i in copies:
            self._refs[i] -= 1
            self._seqs[h][0][j] = self._take()
            dst.append(self._seqs[h][0][j])
        start = []
        for h, c, n in zip(handles, counts, need):
            seq = self._seqs[h]
            seq[0].extend(self._take() for _ in range(n))
            start.append(seq[1])
            seq[1] += c
            if c:
                self._pending.setdefault(h, set()).add(start[-1])
        width = max([1] + [len(self._seqs[h][0]) for h in handles])
        rows = [self._seqs[h][0] + [0] * (width - len(self._seqs[h][0])) for h in handles]
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        positions = [s + i for s, c in zip(start, counts) for i in range(c)]
        B = len(handles)
        # one copy to the device: the table, start, kv_len, cu and positions in turn, and the pages to copy
        flat = [x for r in rows for x in r] + start + [s + c for s, c in zip(start, counts)] + cu + positions
        flat += [i for _, _, i in copies] + dst
        try:
            t = torch.tensor(flat, dtype=torch.int32).to(self.device)
            *t, src, dst_t = t.split([B * width, B, B, B + 1, len(positions), len(copies), len(copies)])
            if copies:
                ops.kv8_copy(self.pages, self.scales, src, dst_t)
        except Exception:  # the pool as it was
            for h, s, c, n in zip(handles, start, counts, need):
                ids = self._seqs[h][0]
                self._release(reversed(ids[len(ids) - n:]))
                del ids[len(ids) - n:]
                self._seqs[h][1] = s
                if c:
                    self._found(self._pending, h, s)
            for (h, j, i), new in zip(reversed(copies), reversed(dst)):
                self._release([new])
                self._seqs[h][0][j] = i
                self._refs[i] += 1
            raise
        for h, j, _ in copies:
            self._moved(h, j * self.page)
        table, start_t, len_t, cu_t, pos = t
        same = B and all(c == counts[0] for c in counts)
        step = Step(table.view(B, width), start_t, len_t, cu_t, pos.view(B, counts[0]) if same else pos, list(counts),
                    list(zip(handles, start, counts)))
        self._uses.add(step.use)
        return step

    def append(self, step, k, v, rope=None, packed=False):
        """The step's new tokens: k / v [B, hk, T, d] where every sequence has T of them, or, packed, [1, hk, rows, d].
        Keys are rotated by their positions when a Rope is given. After a refused append the step's tokens still count:
        append them again, or trim them away; attend refuses sequences that lack them."""
        try:
            self._current(step, new=True)
            for h, s, n in step.spans if self._forked else ():
                if n and any(self._refs[i] > 1 for i in self._seqs[h][0][s // self.page:-(-(s + n) // self.page)]):
                    raise ValueError(f"kv8: sequence {h} shares the pages of this step since it was made")
        except ValueError:  # (tokens that it appended before are there as they were)
            self._lacks(step, lambda h, s: s in self._pending.get(h, ()))
            raise
        try:
            kw = {} if rope is None else {"turns": rope.turns, "layout": rope.layout, "amp": rope.amp}
            if packed:
                if k.shape[2] != sum(step.counts):
                    raise ValueError(f"kv8: {sum(step.counts)} packed rows expected, got {k.shape[2]}")
                kw["cu"] = step.cu
            elif any(c != k.shape[2] for c in step.counts):
                raise ValueError("kv8: sequences with different counts go in packed")
            ops.kv8_append(self.pages, self.scales, k, v, step.table, step.start, **kw)
        except Exception:
            self._lacks(step)
            raise
        for h, s, n in step.spans:
            if n:
                self._found(self._pending, h, s)
                if self._missing:
                    self._found(self._missing, h, s)

    def attend(self, step, q, scale, causal=True, out=None, packed=False):
        """q [B, hq, T, d], the queries of each sequence's last T tokens, over everything cached; or, packed, [1, hq, rows,
        d], the queries of the step's new tokens, for chunks of any and uneven lengths."""
        self._current(step)
        if self._missing:
            for h, s, n in step.spans:
                if any(x < s + n for x in self._missing.get(h, ())):
                    raise ValueError(f"kv8: sequence {h} has tokens that were not appended (their append was refused)")
        if packed:
            if q.shape[2] != sum(step.counts):
                raise ValueError(f"kv8: {sum(step.counts)} packed rows expected, got {q.shape[2]}")
            return ops.kv8_attend_packed(q, self.pages, self.scales, step.table, step.kv_len, step.cu, scale, causal, out)
        return ops.kv8_attend(q, self.pages, self.scales, step.table, step.kv_len, scale, causal, out)


__all__ = ["Cache", "Step"]
