"""Serving-loop bookkeeping: the physical page pool, each request's pages, the batch slots.

The engine derives every decode step's page tables on the device from two things this module
owns on the host: which physical pages a slot's request holds (copied into the slot block
table) and how many tokens it holds.  Three rules of DELTA/Engine/DELTA/scheduler.py decide
both, and are kept exactly:

* Pool order (scheduler.py:8-30): the page ids ``0..n-1`` are shuffled once by a generator
  seeded with ``seed`` (the same permutation ``random.seed(seed); random.shuffle(ids)``
  gives) and handed out from the end of that order.
* Page growth (scheduler.py:60-74): a request starts on one empty page; adding ``n`` tokens
  raises the last page's fill by ``n`` and takes a fresh page each time the fill reaches 16,
  so a full page is always followed by an empty one and ``kv_len = (pages - 1) * 16 + fill``.
* Completion (scheduler.py:83-90): a request ends on a stop token or once prompt plus output
  reach ``max_length``, and its pages go back to the pool.

Requests may share a prefix (``SharedPrefix``: whole pages, computed once) or be forked from one
another: the pages that several hold are counted, and go back to the pool with the last holder.

Everything else is this build's own: requests live in a flat list indexed by id, slots hold
request ids (``None`` when free), waiting ids sit in a deque, and the pool reshuffles its
free ids with its own generator when pages come back (the reference reshuffles with the
process-wide one, so only the order after a release may differ).
"""
from __future__ import annotations

import random
import time
from collections import deque
from typing import Deque, Dict, List, Optional, Sequence, Tuple

import torch

PAGE_SIZE = 16


class PagePool:
    """Shuffled pool of physical KV page ids, with a count of holders for each page that is out."""

    def __init__(self, total_pages: int, seed: Optional[int] = None):
        self.total_pages = int(total_pages)
        self._rng = random.Random(seed)
        ids = list(range(self.total_pages))
        self._rng.shuffle(ids)
        self._free: List[int] = ids          # handed out from the end
        self._held: Dict[int, int] = {}      # page -> holders

    @property
    def available(self) -> int:
        return len(self._free)

    def take(self, n: int = 1) -> List[int]:
        """``n`` pages from the end of the free order (all or none)."""
        if n > len(self._free):
            raise RuntimeError(f"Out of KV pages: {n} wanted, {len(self._free)} free")
        got = [self._free.pop() for _ in range(n)]
        self._held.update((p, 1) for p in got)
        return got

    def share(self, pages: Sequence[int]) -> List[int]:
        """One more holder for each of ``pages``, all of them out; returns them as a list."""
        loose = [p for p in pages if p not in self._held]
        if loose:
            raise RuntimeError(f"page {loose[0]} is not held: it cannot be shared")
        for p in pages:
            self._held[p] += 1
        return list(pages)

    def give_back(self, pages: Sequence[int]) -> None:
        """One holder less for each of ``pages``; those without any are free again."""
        back = []
        for p in pages:
            n = self._held.get(p, 0)
            if n > 1:
                self._held[p] = n - 1
            elif n == 1:
                del self._held[p]
                back.append(p)
        self._free.extend(back)
        self._rng.shuffle(self._free)


class SharedPrefix:
    """The first tokens of several prompts: whole pages, computed when the first of them is served and held until the
    last of them has finished."""

    def __init__(self, tokens: torch.Tensor, pool: PagePool, users: int):
        assert len(tokens) % PAGE_SIZE == 0
        self.tokens = tokens
        self.pages: List[int] = []  # once computed
        self.users = users          # requests that have not finished
        self._pool = pool

    def reserve(self) -> List[int]:
        self.pages = self._pool.take(len(self.tokens) // PAGE_SIZE)
        return self.pages

    def drop(self) -> None:
        """Give the pages back: nobody needs them any more, or they could not be computed."""
        self._pool.give_back(self.pages)
        self.pages = []

    def user_finished(self) -> None:
        self.users -= 1
        if self.users == 0:
            self.drop()


def shared_prefixes(rows: Dict[int, Sequence[int]]) -> Tuple[Dict[int, int], List[List[int]]]:
    """Rows (slot -> pages, in order) that begin with the same pages: each sharing slot's prefix, and the prefixes' pages,
    chosen so that the fewest pages are left to read.

    The rows make a tree of the places where they branch.  A branch at n pages that is taken as a prefix costs n pages once
    and spares n to every row below it that has no deeper one."""
    # (n, rows that go on alone from here, branches below, branch above); a branch comes before those below it
    tree: List[Tuple[int, List[int], List[int], Optional[int]]] = []
    work: List[Tuple[List[int], int, Optional[int]]] = [(sorted(rows), 0, None)]
    while work:
        slots, n, up = work.pop()
        lo, hi = min((rows[s] for s in slots), default=()), max((rows[s] for s in slots), default=())
        most = min(len(lo), len(hi))
        while n < most:  # what the least and the greatest row have in common, all have
            mid = (n + most + 1) // 2
            n, most = (mid, most) if lo[n:mid] == hi[n:mid] else (n, mid - 1)
        by_next: Dict[int, List[int]] = {}
        alone = []
        for s in slots:
            if len(rows[s]) > n:
                by_next.setdefault(rows[s][n], []).append(s)
            else:
                alone.append(s)
        alone += [g[0] for g in by_next.values() if len(g) == 1]
        work += [(g, n, len(tree)) for g in by_next.values() if len(g) > 1]
        if up is not None:
            tree[up][2].append(len(tree))
        tree.append((n, alone, [], up))

    # pages spared below branch v by the pages above that its rows have as their prefix, and whether v is worth taking then
    spared: List[Dict[int, Tuple[int, bool]]] = [{} for _ in tree]
    for v in reversed(range(len(tree))):
        n, alone, below, up = tree[v]
        taken = (len(alone) - 1) * n + sum(spared[c][n][0] for c in below)
        above = {0}
        while up is not None:
            above.add(tree[up][0])
            up = tree[up][3]
        for d in above:
            left = len(alone) * d + sum(spared[c][d][0] for c in below)
            spared[v][d] = max((left, False), (taken, True), key=lambda x: x[0])

    row_prefix: Dict[int, int] = {}
    prefixes: List[List[int]] = []
    inherited: List[Tuple[int, int]] = []  # each branch's (pages, prefix) for the rows that have no deeper one
    for v, (n, alone, below, up) in enumerate(tree):
        d, group = inherited[up] if up is not None else (0, -1)
        if spared[v][d][1]:
            d, group = n, len(prefixes)
            first = v
            while not tree[first][1]:
                first = tree[first][2][0]
            prefixes.append(list(rows[tree[first][1][0]][:n]))
        inherited.append((d, group))
        if group >= 0:
            row_prefix.update((s, group) for s in alone)
    return row_prefix, prefixes


class ServingRequest:
    """One prompt being served: its tokens, its pages and its timing."""

    WAITING, ACTIVE, FINISHED = "waiting", "active", "finished"

    def __init__(self, rid: int, prompt: torch.Tensor, max_length: int, stop_ids: Sequence[int],
                 pool: PagePool, prefix: Optional[SharedPrefix] = None):
        self.rid = rid
        self.prompt = prompt
        self.max_length = int(max_length)
        self.stop_ids = set(int(t) for t in stop_ids)
        self.generated: List[int] = []
        self.pages: List[int] = []
        self.fill = 0                  # tokens in the last page
        self.state = self.WAITING
        self.t_start: Optional[float] = None
        self.t_end: Optional[float] = None
        self.prefix = prefix           # whose tokens the prompt begins with
        self.cached = 0                # prompt tokens that were in the cache when serving began
        self._pool = pool

    # -- pages
    def admit(self) -> None:
        """Start serving: one empty page, behind the pages of the prefix (computed by now) if there is one."""
        own = self._pool.take(1)
        self.state = self.ACTIVE
        self.t_start = time.perf_counter()
        self.pages = own
        self.fill = 0
        if self.prefix is not None:
            self.pages = self._pool.share(self.prefix.pages) + own
            self.cached = len(self.prefix.tokens)

    def fork(self, rid: int, more: torch.Tensor, max_length: int, stop_ids: Sequence[int]) -> "ServingRequest":
        """A request that continues this one's tokens so far with ``more``, already being served: it shares the full
        pages and has a page of its own for the ``fill`` tokens of the last one (copied by the caller)."""
        prompt = self.prompt.to(torch.long)
        prompt = torch.cat([prompt, torch.tensor(self.generated, dtype=torch.long, device=prompt.device),
                            more.to(prompt.device, torch.long)])
        child = ServingRequest(rid, prompt, max_length, stop_ids, self._pool)
        own = self._pool.take(1)
        child.state = self.ACTIVE
        child.t_start = time.perf_counter()
        child.pages = self._pool.share(self.pages[:-1]) + own
        child.fill = self.fill
        child.cached = self.kv_len()
        return child

    def reserve(self, n_tokens: int, page_size: int = PAGE_SIZE) -> None:
        """Account for ``n_tokens`` new tokens (the page-growth rule above)."""
        self.fill += int(n_tokens)
        grow = self.fill // page_size
        if grow:
            self.pages.extend(self._pool.take(grow))
            self.fill -= grow * page_size

    def kv_len(self, page_size: int = PAGE_SIZE) -> int:
        return (len(self.pages) - 1) * page_size + self.fill

    # -- tokens
    def next_input(self) -> torch.Tensor:
        """The tokens of this request's next forward: the prompt's that are not cached, then the last output."""
        return self.prompt[self.cached:] if not self.generated else torch.tensor([self.generated[-1]], dtype=torch.long)

    def record(self, token: int) -> bool:
        """Append an output token; True when the request is now finished."""
        self.generated.append(int(token))
        if int(token) in self.stop_ids or len(self.prompt) + len(self.generated) >= self.max_length:
            self.finish()
            return True
        return False

    def finish(self) -> None:
        """End serving: the pages go back to the pool."""
        self._pool.give_back(self.pages)
        if self.prefix is not None:
            self.prefix.user_finished()
        self.state = self.FINISHED
        self.t_end = time.perf_counter()

    @property
    def finished(self) -> bool:
        return self.state == self.FINISHED

    def summary(self, tokenizer=None) -> Dict:
        """The per-request record the reference's result consumers read (same keys)."""
        elapsed = (self.t_end - self.t_start) if (self.t_end and self.t_start) else 0
        n_out = len(self.generated)
        rec = {"request_id": self.rid, "status": self.state, "input_length": len(self.prompt),
               "output_length": n_out, "tokens_generated": n_out, "total_time": elapsed,
               "tokens_per_second": n_out / elapsed if elapsed > 0 else 0}
        if tokenizer is not None:
            rec["input_text"] = _decode_or_placeholder(tokenizer, self.prompt)
            rec["output_text"] = _decode_or_placeholder(tokenizer, self.generated)
        return rec


def _decode_or_placeholder(tokenizer, ids) -> str:
    try:
        return tokenizer.decode(ids, skip_special_tokens=True)
    except Exception:  # a tokenizer that cannot take these ids still yields a record
        return f"[{len(ids)} tokens]"


class BatchSlots:
    """Fixed batch slots over a queue of requests (free slots take waiting requests in order)."""

    def __init__(self, batch_size: int, pool: PagePool, verbose: bool = True):
        self.pool = pool
        self.verbose = verbose
        self.slots: List[Optional[int]] = [None] * int(batch_size)
        self.requests: List[ServingRequest] = []
        self.waiting: Deque[int] = deque()
        self.tokens_generated = 0
        self.t_start: Optional[float] = None

    def submit(self, prompts: Sequence[torch.Tensor], max_lengths, stop_ids: Sequence[int],
               prefix_tokens: Optional[torch.Tensor] = None) -> None:
        """Queue requests; with ``prefix_tokens`` each prompt continues them, and their whole pages (short of the last
        token of a prompt that adds none: every request feeds at least one token of its own) are shared."""
        prefix = None
        if prefix_tokens is not None and len(prompts):
            prefix_tokens = prefix_tokens.to(torch.long)
            prompts = [torch.cat([prefix_tokens.to(p.device), p.to(torch.long)]) for p in prompts]
            whole = min(len(prefix_tokens), min(len(p) for p in prompts) - 1) // PAGE_SIZE * PAGE_SIZE
            if whole > 0:
                prefix = SharedPrefix(prefix_tokens[:whole], self.pool, len(prompts))
        for i, prompt in enumerate(prompts):
            cap = max_lengths[i] if isinstance(max_lengths, (list, tuple)) else max_lengths
            req = ServingRequest(len(self.requests), prompt, cap, stop_ids, self.pool, prefix)
            self.requests.append(req)
            self.waiting.append(req.rid)
        if self.verbose:
            print(f"queued {len(prompts)} request(s); {len(self.waiting)} waiting")

    def fill_free_slots(self) -> List[Tuple[int, ServingRequest]]:
        """Place waiting requests into free slots (lowest slot first); returns (slot, request)."""
        placed = []
        for s, rid in enumerate(self.slots):
            if rid is None and self.waiting:
                req = self.requests[self.waiting.popleft()]
                self.slots[s] = req.rid
                placed.append((s, req))
        return placed

    def unplace(self, placed: Sequence[Tuple[int, ServingRequest]]) -> None:
        """Requests of ``fill_free_slots`` that could not be admitted go back to the head of the queue."""
        for s, req in reversed(placed):
            self.slots[s] = None
            self.waiting.appendleft(req.rid)

    def place(self, req: ServingRequest) -> int:
        """Put an already served request (a fork) into a free slot."""
        slot = self.free_slot()
        if slot is None:
            raise RuntimeError("no free slot")
        self.requests.append(req)
        self.slots[slot] = req.rid
        return slot

    def free_slot(self) -> Optional[int]:
        return next((s for s, rid in enumerate(self.slots) if rid is None), None)

    def release_finished(self) -> List[int]:
        """Free the slots whose request finished; returns those slot ids."""
        done = [s for s, rid in enumerate(self.slots) if rid is not None and self.requests[rid].finished]
        for s in done:
            self.slots[s] = None
        return done

    def occupied(self) -> List[int]:
        return [s for s, rid in enumerate(self.slots) if rid is not None]

    def request_in(self, slot: int) -> ServingRequest:
        return self.requests[self.slots[slot]]

    def any_active(self) -> bool:
        return any(rid is not None for rid in self.slots)

    def report(self, tokenizer=None) -> List[Dict]:
        return [r.summary(tokenizer) for r in self.requests if r.finished]
