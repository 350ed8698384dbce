"""A paged K/V cache: which pages each sequence has, and the tensors they are in.

``PagePool`` keeps the books on the host: sequences are lists of page ids,
pages are counted, and forked sequences share theirs until one of them writes.
``PagedCache`` adds the tensors ([layers, pages, kv_heads, page_size, d]) and
runs the copies its pool asks for; ``nkilab.ops`` writes to them and attends
over them, ``nkilab.model.nki_decode`` runs a decoder block over them.  The
reference has no cache (its block attends over one prompt, model.py:59-67).

    cache = PagedCache(pages=1024, kv_heads=8, head_dim=128, layers=24)
    seq = cache.add()
    step = cache.step([seq], [len(prompt)])        # rows for the prompt
    x = nki_decode(block, x, cache, step, layer)   # for every layer
    step = cache.step([seq], [16], tree=[parents]) # a tree of 16 drafted tokens
    ...
    cache.accept(step, [[0, 3, 7]])                # the path that was accepted
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops


class OutOfPages(RuntimeError):
    """No free page is left for what was asked; nothing has changed."""


class PagePool:
    """Pages and sequences, on the host."""

    def __init__(self, pages: int, page_size: int):
        if pages < 1 or page_size < 1:
            raise ValueError(f"PagePool: pages={pages} and page_size={page_size} must be at least 1")
        self.pages, self.page_size = int(pages), int(page_size)
        self._free = list(range(self.pages - 1, -1, -1))  # taken from the end: the lowest first
        self._users = [0] * self.pages
        self._tables: dict[int, list[int]] = {}
        self._lens: dict[int, int] = {}
        self._floor: dict[int, int] = {}  # the length a sequence had when it last gave up pages
        self._next = 0
        # Counts what happens to sequences; and its values when each last changed
        # its length, and when rows or pages of it last went.
        self._clock = 0
        self._resized: dict[int, int] = {}
        self._cut: dict[int, int] = {}

    def _note(self, when: dict[int, int], seq: int) -> None:
        self._clock += 1
        when[seq] = self._clock

    def add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._tables[seq], self._lens[seq], self._floor[seq] = [], 0, 0
        self._resized[seq] = self._cut[seq] = self._clock
        return seq

    def length(self, seq: int) -> int:
        return self._lens[seq]

    def pages_of(self, seq: int) -> list[int]:
        """The sequence's pages in order; -1 where one was released."""
        return list(self._tables[seq])

    def free_pages(self) -> int:
        return len(self._free)

    def _drop(self, page: int) -> None:
        if page < 0:
            return
        self._users[page] -= 1
        if self._users[page] == 0:
            self._free.append(page)

    def fork(self, seq: int) -> int:
        """A sequence with the same rows, in the same pages until either writes (rows
        that a step has yet to bring are copied as they are)."""
        table = list(self._tables[seq])
        new = self.add()
        self._tables[new], self._lens[new] = table, self._lens[seq]
        self._floor[new] = self._floor[seq]
        for p in self._tables[new]:
            if p >= 0:
                self._users[p] += 1
        return new

    def free(self, seq: int) -> None:
        """Ends a sequence; pages that no other has are free again."""
        for p in self._tables.pop(seq):
            self._drop(p)
        del self._lens[seq], self._floor[seq], self._resized[seq], self._cut[seq]
        self._clock += 1

    def _plan(self, seqs: list[int], starts: list[int], ends: list[int], keep: bool = False) -> "_Plan":
        """What `own` will do; nothing changes."""
        ps = self.page_size
        if len(set(seqs)) != len(seqs):
            raise ValueError(f"a sequence is named twice: {seqs}")
        users = dict()  # pages' users as they will be
        wanted = []     # (sequence, place in its table, the page that is there and to be kept)
        for seq, start, end in zip(seqs, starts, ends):
            table = self._tables[seq]
            for i in range(start // ps, -(-end // ps) if end > start else 0):
                if i >= len(table):
                    wanted.append((seq, i, None))
                    continue
                p = table[i]
                if p < 0:
                    raise ValueError(f"sequence {seq}: rows {i * ps} .. were released")
                left = users.get(p, self._users[p])
                if left > 1:
                    wanted.append((seq, i, p if keep or i * ps < start else None))
                    users[p] = left - 1
        if len(wanted) > len(self._free):
            raise OutOfPages(f"{len(wanted)} pages needed, {len(self._free)} of {self.pages} free")
        new = self._free[len(self._free) - len(wanted):][::-1]  # from the end
        return _Plan([(seq, i, page) for (seq, i, _), page in zip(wanted, new)],
                     [(old, page) for (_, _, old), page in zip(wanted, new) if old is not None],
                     {seq: max(end, 0) for seq, end in zip(seqs, ends)})

    def _planned(self, plan: "_Plan") -> dict[int, list[int]]:
        """The tables of the plan's sequences as they will be."""
        tables = {seq: list(self._tables[seq]) for seq in plan.lens}
        for seq, i, page in plan.pages:
            tables[seq][i:i + 1] = [page]
        return tables

    def _apply(self, plan: "_Plan") -> None:
        del self._free[len(self._free) - len(plan.pages):]
        for seq, i, page in plan.pages:
            self._users[page] = 1
            table = self._tables[seq]
            if i < len(table):
                self._users[table[i]] -= 1
                self._note(self._cut, seq)
            table[i:i + 1] = [page]
        for seq, n in plan.lens.items():
            if n != self._lens[seq]:
                self._lens[seq] = n
                self._note(self._resized, seq)

    def own(self, seqs: list[int], starts: list[int], ends: list[int], keep: bool = False) -> list[tuple[int, int]]:
        """Gives each sequence pages of its own for rows starts[i] .. ends[i] - 1 and
        that length.  Returns the (from, to) copies that are to be made first; the
        rows before starts[i] are kept, those from there on with `keep` only."""
        plan = self._plan(seqs, starts, ends, keep)
        self._apply(plan)
        return plan.copies

    def trim(self, seq: int, length: int) -> None:
        """Cuts a sequence to its first `length` rows (no fewer than it had when
        pages were last released: its next tokens would look for them)."""
        if not self._floor[seq] <= length <= self._lens[seq]:
            raise ValueError(f"sequence {seq}: length {length} outside [{self._floor[seq]}, {self._lens[seq]}]")
        table = self._tables[seq]
        while len(table) > -(-length // self.page_size):
            self._drop(table.pop())
        if length < self._lens[seq]:
            self._note(self._resized, seq)
            self._note(self._cut, seq)
        self._lens[seq] = length

    def release(self, seq: int, window: int, sinks: int = 0) -> int:
        """Gives up the pages that no later token sees under a window: those whose
        rows are all at least `window` before the sequence's next position and
        none of the first `sinks`.  Returns how many.  (Tokens before the next may
        see more: it is called once the latest step has been run.)"""
        if window < 1 or sinks < 0:
            raise ValueError(f"window={window} must be at least 1 and sinks={sinks} at least 0")
        ps, table, n = self.page_size, self._tables[seq], 0
        for i in range(-(-sinks // ps), max(0, (self._lens[seq] - window + 1) // ps)):
            if table[i] >= 0:
                self._drop(table[i])
                table[i] = -1
                n += 1
        if n:
            self._floor[seq] = self._lens[seq]
            self._note(self._cut, seq)
        return n

    def _moves(self) -> dict[int, int]:
        """The copies of a compaction: every page in use that is not among the lowest, to the lowest free ones."""
        used = [p for p in range(self.pages) if self._users[p]]
        low = [p for p in range(len(used)) if not self._users[p]]
        return dict(zip([p for p in used if p >= len(used)], low))

    def _rename(self, moves: dict[int, int]) -> None:
        for table in self._tables.values():
            table[:] = [moves.get(p, p) for p in table]
        for a, b in moves.items():
            self._users[b], self._users[a] = self._users[a], 0
        self._free = [p for p in range(self.pages - 1, -1, -1) if not self._users[p]]

    def compact(self) -> list[tuple[int, int]]:
        """Moves the pages in use to the lowest ids.  Returns the copies."""
        moves = self._moves()
        self._rename(moves)
        return list(moves.items())


@dataclass
class _Plan:
    """Pages that sequences are to be given, decided before anything changes."""
    pages: list[tuple[int, int, int]]  # (sequence, place in its table, page), in the order that they are taken
    copies: list[tuple[int, int]]      # (from, to), made before the plan is applied
    lens: dict[int, int]


def _depth(parents: list[int]) -> int:
    """Nodes of a tree's longest branch."""
    depths = []
    for p in parents:
        depths.append(1 + (depths[p] if p >= 0 else 0))
    return max(depths, default=0)


@dataclass
class CacheStep:
    """The new rows of some sequences, as the operators take them (device
    tensors), and as the cache knows them."""
    seqs: list[int]
    counts: list[int]
    table: torch.Tensor      # int32 [batch, columns]
    lens: torch.Tensor       # int32 [batch], with the new rows
    q_start: torch.Tensor    # int32 [batch + 1]
    max_q: int
    tree: torch.Tensor | None     # mask words, as ops.tree_mask has them without a window
    parents: torch.Tensor | None  # the trees' parents, packed
    depth: int                    # nodes of the longest branch
    resized: list[int]       # when the cache last changed the sequences' lengths,
    cut: list[int]           # when it last took rows or pages from them,
    moved: int               # how often it had been compacted,
    checked: int             # and when the step last stood

    @property
    def rows(self) -> int:
        return sum(self.counts)


class PagedCache(PagePool):
    """K and V of every layer in pages, and the sequences they belong to."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, layers: int = 1, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str | None = None):
        super().__init__(pages, page_size)
        shape = (layers, pages, kv_heads, page_size, head_dim)
        device = torch.device("cuda") if device is None else device
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self._moved = 0

    def _copy(self, copies: list[tuple[int, int]]) -> None:
        if copies:
            ops.cache_copy_pages(self.k, self.v, copies)

    def _tensor(self, rows) -> torch.Tensor:
        return torch.tensor(rows, dtype=torch.int32).to(self.k.device)

    def step(self, seqs: list[int], counts: list[int], tree: list[list[int]] | None = None) -> CacheStep:
        """Makes room for counts[i] new rows of sequence seqs[i] (shared pages that
        they touch are copied) and describes them.  tree: each sequence's drafted
        tree as its nodes' parents (see ``ops.tree_mask``).  A step stands, also
        when later ones are made, until one of its sequences ends or gives up
        rows or pages, or pages are moved; calls with it are refused from then on."""
        seqs, counts = list(seqs), [int(n) for n in counts]
        if len(seqs) != len(counts) or any(n < 0 for n in counts):
            raise ValueError(f"step: {len(seqs)} sequences and counts {counts}")
        if tree is not None and [len(p) for p in tree] != counts:
            raise ValueError(f"step: trees of {[len(p) for p in tree]} nodes for counts {counts}")
        for t in tree or []:
            if not all(-1 <= p < i for i, p in enumerate(t)):
                raise ValueError(f"step: parents {t} must be nodes before their own, or -1")
        old = [self._lens[s] for s in seqs]
        ends = [a + n for a, n in zip(old, counts)]
        # The books change once everything that may be refused is done.
        plan = self._plan(seqs, old, ends)
        tables = self._planned(plan)
        self._copy(plan.copies)
        width = max([len(tables[s]) for s in seqs] + [1])
        start = [0]
        for n in counts:
            start.append(start[-1] + n)
        # One upload: the table's rows, the lengths, the offsets.
        flat = []
        for s in seqs:
            flat += tables[s] + [-1] * (width - len(tables[s]))
        B, nt = len(seqs), len(flat)
        dev = self._tensor(flat + ends + start + ([p for t in tree for p in t] if tree else []))
        step = CacheStep(seqs, counts, dev[:nt].view(B, width), dev[nt:nt + B], dev[nt + B:nt + 2 * B + 1],
                         max(counts + [0]), None, None, 0, [], [], self._moved, 0)
        if tree is not None:
            step.parents = dev[nt + 2 * B + 1:]
            step.depth = max(map(_depth, tree), default=0)
            step.tree = ops.tree_mask(step.parents, q_start=step.q_start, max_q=step.max_q)
        self._apply(plan)
        step.resized, step.cut, step.checked = ([self._resized[s] for s in seqs], [self._cut[s] for s in seqs], self._clock)
        return step

    def _check(self, fn: str, step: CacheStep) -> None:
        """The step's rows are where its table has them, in pages of its sequences' own."""
        if step.checked == self._clock:
            return  # (nothing has happened since it last stood)
        self._check_moved(fn, step)
        for s, at in zip(step.seqs, step.cut):
            if self._cut.get(s) != at:
                raise ValueError(f"{fn}: the step's table is stale, sequence {s} has ended or given up rows or pages since")
        step.checked = self._clock

    def _check_moved(self, fn: str, step: CacheStep) -> None:
        if step.moved != self._moved:
            raise ValueError(f"{fn}: the step's table is stale, the cache has been compacted since")

    def accept(self, step: CacheStep, paths: list[list[int]]) -> None:
        """Keeps the accepted path of each sequence's rows of `step` (its latest),
        strictly ascending nodes, and drops the others.  Once for a step."""
        paths = [[int(i) for i in p] for p in paths]
        if len(paths) != len(step.seqs):
            raise ValueError(f"accept: {len(paths)} paths for {len(step.seqs)} sequences")
        for s, n, path in zip(step.seqs, step.counts, paths):
            if any(a >= b for a, b in zip([-1] + path, path + [n])):
                raise ValueError(f"accept: path {path} does not ascend within [0, {n})")
        self._check_moved("accept", step)
        for s, at in zip(step.seqs, step.resized):
            if self._resized.get(s) != at:
                raise ValueError(f"accept: sequence {s} has ended, or changed its length since: not its latest step")
        lens = [self._lens[s] for s in step.seqs]
        ctx = [a - n for a, n in zip(lens, step.counts)]
        for s, c, path in zip(step.seqs, ctx, paths):
            if c + len(path) < self._floor[s]:
                raise ValueError(f"accept: sequence {s} gave up pages at length {self._floor[s]}, the path leaves "
                                 f"{c + len(path)}; release pages after a path is accepted")
        stay = [sum(i == node for i, node in enumerate(p)) for p in paths]  # (an ascending path's first: in place already)
        if any(m < len(p) for m, p in zip(stay, paths)):
            table = step.table
            # Pages of its own for the rows that move; those that they come from are only read.
            plan = self._plan(step.seqs, [c + m for c, m in zip(ctx, stay)], [c + len(p) for c, p in zip(ctx, paths)],
                              keep=True)
            plan.lens = dict(zip(step.seqs, lens))  # (until the others are dropped)
            if plan.copies or any(self._cut[s] != at for s, at in zip(step.seqs, step.cut)):  # forked since the step
                self._copy(plan.copies)
                rows = self._planned(plan)
                table = self._tensor([rows[s] + [-1] * (table.shape[1] - len(rows[s])) for s in step.seqs])
            width = max(len(p) for p in paths)
            ops.cache_accept(self.k, self.v, table, step.lens,
                             self._tensor([p + [-1] * (width - len(p)) for p in paths]), q_start=step.q_start)
            self._apply(plan)
        for s, n, c, path in zip(step.seqs, step.counts, ctx, paths):
            self.trim(s, c + len(path))
            if n:  # (once, also where the whole of it is accepted)
                self._note(self._resized, s)

    def compact(self) -> list[tuple[int, int]]:
        """Moves the pages in use to the lowest ids, so that the others are one
        stretch at the end.  Steps made before a move are refused from then on."""
        moves = self._moves()
        self._copy(list(moves.items()))
        self._rename(moves)
        self._moved += bool(moves)
        self._clock += 1
        return list(moves.items())

    def append(self, layer: int, step: CacheStep, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None, rope_base: float | None = None) -> None:
        """``ops.cache_append_into`` of the step's rows in a layer."""
        self._check("append", step)
        ops.cache_append_into(k, v, self.k[layer], self.v[layer], step.table, step.lens, step.q_start, step.max_q,
                              step.tree, q, q_out, rope_base)

    def attention_into(self, layer: int, step: CacheStep, q: torch.Tensor, o: torch.Tensor, window: int | None = None,
                       sinks: int = 0, scale: float | None = None) -> torch.Tensor:
        """``ops.paged_attention_into`` of the step's rows in a layer.  A drafted
        node sees its branch as the row of a prompt would: under a window, the
        ancestors within it and the sinks."""
        self._check("attention_into", step)
        tree = step.tree
        if tree is not None and window is not None and step.depth > window:
            tree = ops.tree_mask(step.parents, step.q_start, step.max_q, window=window, sinks=sinks, lens=step.lens)
        return ops.paged_attention_into(q, o, self.k[layer], self.v[layer], step.table, step.lens, step.q_start,
                                        step.max_q, window, sinks, tree, scale)
