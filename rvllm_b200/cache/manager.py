"""The cache manager: paged keys and values with a block table per request and cache group,
and slots of fixed-size per-request state.

Layers whose mixers need the same thing (same kv heads, head size and window) form a group; a
group has its own pages, its own block table per request and one device tensor
[cache slots of the group, num_pages, planes (2: k, v; 1: one shared row), kv_heads, page_size, head_dim].  A page id
addresses the same page in every slot of its group.  Pages are handed out when tokens are about
to be written into them and come back when the request ends, is pre-empted, or - for a window
group - when every later query is past them.  The block table keeps -1 where a page was
given back.  Every request also holds one state slot; mixers with `StateNeed` get a tensor
[max_seqs, *shape] that is zeroed when the slot is handed to a new request.

A group whose values are not as wide as its keys (`KvCacheNeed.value_dim`) keeps its pages flat:
[cache slots, num_pages, kv_heads * page_size * (head_dim + value_dim)], a page's key rows first, then its
value rows.  A chunk group (`KvCacheNeed.chunk`) gives a page back once the block of positions that the next
query lies in starts above it.  A cache slot whose mixer is made of several mixers (`CompositeNeed`) has one
sub-view per member, each handled as a cache slot of its own.

Requests that begin with the same tokens can hold the same pages (`share`), where every group keeps all keys and no layer
has state of fixed size: a page whose tokens are all known to be the same and computed is taken over, what follows is the
request's own.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, Hashable, List, Optional, Tuple

import torch

from ..errors import KvExhausted, SchedulerError
from ..parts.base import CompositeNeed, KvCacheNeed, StateNeed
from .pools import PagePool, SlotPool


@dataclass
class CacheView:
    """What a mixer sees of its cache slot."""
    group: Optional[int]                 # index of the page group (None: no pages)
    kv: Optional[torch.Tensor]           # [num_pages, planes, kv_heads, page_size, head_dim] (flat pages: [num_pages, elements])
    state: Optional[torch.Tensor] = None  # [max_seqs, *shape]
    parts: Tuple["CacheView", ...] = ()   # one view per member of a mixer made of several mixers


@dataclass
class _Group:
    need: KvCacheNeed
    cache_slots: List[int]
    pool: PagePool
    tensor: Optional[torch.Tensor] = None


@dataclass
class _Request:
    state_slot: int
    num_tokens: int = 0
    tables: List[List[int]] = field(default_factory=list)   # per group: page of each logical block, -1 if freed
    first_live: List[int] = field(default_factory=list)     # per group: first logical block still held
    on_device: List[int] = field(default_factory=list)      # per group: blocks that the step function's table on the device has


def flat_needs(needs: Dict[int, object]) -> Dict[object, object]:
    """cache slot -> need, with the members of a `CompositeNeed` under the keys (slot, member index)."""
    out: Dict[object, object] = {}
    for slot in sorted(needs):
        need = needs[slot]
        if isinstance(need, CompositeNeed):
            for i, member in enumerate(need.parts):
                out[(slot, i)] = member
        else:
            out[slot] = need
    return out


class CacheManager:
    def __init__(self, needs: Dict[int, object], num_pages: int, page_size: int, max_seqs: int,
                 dtype: torch.dtype = torch.float32, device="cpu", allocate: bool = True):
        self.page_size, self.num_pages, self.max_seqs = page_size, num_pages, max_seqs
        self.dtype, self.device = dtype, device
        self.groups: List[_Group] = []
        self._slot_group: Dict[object, int] = {}
        self._slot_index: Dict[object, int] = {}
        self._state: Dict[object, torch.Tensor] = {}
        self._state_needs: Dict[object, StateNeed] = {}
        self._members = {slot: len(need.parts) for slot, need in needs.items() if isinstance(need, CompositeNeed)}
        for slot, need in flat_needs(needs).items():
            if isinstance(need, KvCacheNeed):
                for gi, g in enumerate(self.groups):
                    if g.need == need:
                        break
                else:
                    gi = len(self.groups)
                    self.groups.append(_Group(need, [], PagePool(num_pages)))
                self._slot_group[slot] = gi
                self._slot_index[slot] = len(self.groups[gi].cache_slots)
                self.groups[gi].cache_slots.append(slot)
            elif isinstance(need, StateNeed):
                self._state_needs[slot] = need
            elif need is not None:
                raise SchedulerError(f"cache slot {slot}: unknown kind of need {need!r}")
        self.slots = SlotPool(max_seqs)
        self._has_window = any(g.need.window is not None or g.need.chunk is not None for g in self.groups)
        self.requests: Dict[Hashable, _Request] = {}
        self.changes = 0               # how often a request came, went or took over pages
        if allocate:
            for g in self.groups:
                if g.need.flat_pages:
                    shape = (len(g.cache_slots), num_pages, g.need.num_kv_heads * page_size * g.need.row_elements)
                else:
                    shape = (len(g.cache_slots), num_pages, g.need.planes, g.need.num_kv_heads, page_size, g.need.head_dim)
                g.tensor = torch.zeros(shape, dtype=dtype, device=device)
            for slot, need in self._state_needs.items():
                self._state[slot] = torch.zeros((max_seqs, *need.shape), dtype=getattr(torch, need.dtype), device=device)

    # ---- sizes ------------------------------------------------------------------------------
    @staticmethod
    def bytes_per_page(needs: Dict[int, object], page_size: int, dtype: torch.dtype) -> int:
        """Bytes that one more page per group costs over all cache slots."""
        el = torch.empty((), dtype=dtype).element_size()
        return sum(n.num_kv_heads * page_size * n.row_elements * el for n in flat_needs(needs).values() if isinstance(n, KvCacheNeed))

    @staticmethod
    def state_bytes_per_request(needs: Dict[int, object]) -> int:
        """Bytes of fixed-size state that one request slot holds over all cache slots."""
        total = 0
        for n in flat_needs(needs).values():
            if isinstance(n, StateNeed):
                count = 1
                for d in n.shape:
                    count *= d
                total += count * torch.empty((), dtype=getattr(torch, n.dtype)).element_size()
        return total

    def view(self, cache_slot) -> CacheView:
        if cache_slot in self._members:
            return CacheView(None, None, None, tuple(self.view((cache_slot, i)) for i in range(self._members[cache_slot])))
        gi = self._slot_group.get(cache_slot)
        kv = None
        if gi is not None and self.groups[gi].tensor is not None:
            kv = self.groups[gi].tensor[self._slot_index[cache_slot]]
        return CacheView(gi, kv, self._state.get(cache_slot))

    def blocks_for(self, num_tokens: int) -> int:
        return (num_tokens + self.page_size - 1) // self.page_size

    def peak_pages(self, num_tokens: int, largest_portion: int) -> List[int]:
        """Per group, the most pages a request of `num_tokens` tokens holds at any one time when no
        step brings it more than `largest_portion` tokens.  A group that keeps every key needs the
        pages of all its tokens; a window group holds the window behind the first token of a step
        plus the step's own tokens (what lies below is given back after each step)."""
        out = []
        for g in self.groups:
            full = self.blocks_for(num_tokens)
            w = g.need.window if g.need.window is not None else g.need.chunk
            if w is None:
                out.append(full)
            else:
                # keys [first - w + 1, first + portion) straddle at most one page more than their count fills
                out.append(min(full, self.blocks_for(w - 1 + max(1, largest_portion)) + 1))
        return out

    # ---- requests ---------------------------------------------------------------------------
    def has(self, req: Hashable) -> bool:
        return req in self.requests

    def admit(self, req: Hashable) -> int:
        if req in self.requests:
            raise SchedulerError(f"request {req!r} is already in the cache")
        slot = self.slots.allocate(req)
        self.changes += 1
        self.requests[req] = _Request(slot, 0, [[] for _ in self.groups], [0 for _ in self.groups], [0 for _ in self.groups])
        for t in self._state.values():
            t[slot].zero_()
        return slot

    @property
    def can_share(self) -> bool:
        """True where a request's first pages say all there is to know about its first tokens."""
        return bool(self.groups) and not self._has_window and not self._state_needs

    @property
    def any_shared(self) -> bool:
        """Whether any page has several holders."""
        return self.can_share and self.groups[0].pool.any_shared

    def share(self, req: Hashable, donor: Hashable, num_tokens: int) -> None:
        """The pages of `donor`'s first `num_tokens` tokens (a multiple of the page size) become the first pages of `req`, which has
        none yet.  The caller knows that both begin with these tokens and that the donor's are in the cache."""
        r, d = self.requests[req], self.requests[donor]
        if not self.can_share:
            raise SchedulerError("pages cannot be shared: a layer has a window, a chunk or state of its own")
        if r.num_tokens or any(r.tables):
            raise SchedulerError(f"request {req!r} has tokens already")
        if num_tokens < 1 or num_tokens % self.page_size or num_tokens > d.num_tokens:
            raise SchedulerError(f"request {req!r}: {num_tokens} tokens of {donor!r} cannot be shared: it has {d.num_tokens}, in pages of {self.page_size}")
        self.changes += 1
        n = num_tokens // self.page_size
        for g, mine, theirs in zip(self.groups, r.tables, d.tables):
            g.pool.share(theirs[:n], req)
            mine.extend(theirs[:n])
        r.num_tokens = num_tokens

    def shared_groups(self, reqs) -> List[Tuple[List[int], int]]:
        """Which of the requests `reqs` begin with the same pages: (places in `reqs`, tokens) per group, each request in one group at
        most.  Where a few of those that share a beginning share more among themselves, the grouping that saves the most keys is taken
        (looked for up to 64 beginnings within one another)."""
        if not self.any_shared:
            return []
        tables = [self.requests[r].tables[0] for r in reqs]

        def grouped(members: List[int], depth: int, inside: int = 0):
            """(keys saved, groups) of requests whose first `depth` pages are the same"""
            if len(members) < 2:
                return 0, []
            first = tables[members[0]]
            common = min(len(tables[m]) for m in members)
            run = first[depth:common]                # whole runs of pages are compared at a time
            for m in members[1:]:
                t, lo = tables[m], depth
                if t[lo:common] == run:
                    continue
                while lo < common:
                    mid = (lo + common) // 2
                    if t[lo:mid + 1] == first[lo:mid + 1]:
                        lo = mid + 1
                    else:
                        common = mid
                run = first[depth:common]
            parts: Dict[int, List[int]] = {}
            for m in members:
                if len(tables[m]) > common:
                    parts.setdefault(tables[m][common], []).append(m)
            saved, groups = (len(members) - 1) * common * self.page_size, [(members, common * self.page_size)] if common else []
            deeper = [grouped(ms, common, inside + 1) for ms in parts.values() if len(ms) > 1 and inside < 64]
            if sum(d[0] for d in deeper) > saved:
                return sum(d[0] for d in deeper), [g for d in deeper for g in d[1]]
            return saved, groups
        return grouped(list(range(len(tables))), 0)[1]

    def num_tokens(self, req: Hashable) -> int:
        return self.requests[req].num_tokens

    def state_slot(self, req: Hashable) -> int:
        return self.requests[req].state_slot

    def pages_needed(self, req: Optional[Hashable], n_new: int, have_tokens: Optional[int] = None) -> List[int]:
        """New pages per group that appending `n_new` tokens would take."""
        if req is not None and req in self.requests:
            r = self.requests[req]
            return [self.blocks_for(r.num_tokens + n_new) - len(t) for t in r.tables]
        have = have_tokens or 0
        return [self.blocks_for(have + n_new) - self.blocks_for(have) for _ in self.groups]

    def can_append(self, req: Optional[Hashable], n_new: int, reserved: Optional[List[int]] = None) -> bool:
        need = self.pages_needed(req, n_new)
        res = reserved or [0] * len(self.groups)
        return all(n + r <= g.pool.num_free for n, r, g in zip(need, res, self.groups))

    def append(self, req: Hashable, n_new: int) -> int:
        """Reserve room for `n_new` more tokens; returns the position of the first.  Takes every
        page it needs or none (`KvExhausted`)."""
        r = self.requests[req]
        blocks = (r.num_tokens + n_new + self.page_size - 1) // self.page_size
        need = [blocks - len(t) for t in r.tables]
        if any(need):
            for n, g in zip(need, self.groups):
                if n > g.pool.num_free:
                    raise KvExhausted(n, g.pool.num_free, f"request {req!r}")
            for n, g, table in zip(need, self.groups, r.tables):
                if n > 0:
                    table.extend(g.pool.allocate(n, req))
        start = r.num_tokens
        r.num_tokens += n_new
        return start

    def block_table(self, req: Hashable, group: int) -> List[int]:
        return self.requests[req].tables[group]

    def slot_mapping(self, req: Hashable, group: int, start: int, n: int) -> List[int]:
        table = self.requests[req].tables[group]
        ps = self.page_size
        out = []
        for pos in range(start, start + n):
            page = table[pos // ps]
            if page < 0:
                raise SchedulerError(f"request {req!r}: position {pos} lies in a page that was given back")
            out.append(page * ps + pos % ps)
        return out

    def release_passed(self, req: Hashable) -> int:
        """Give back the pages of window and chunk groups that no later query can see.  The next query
        sits at position >= num_tokens and sees keys > position - window, and - in a chunk group - no key
        below the start of its own block of `chunk` positions."""
        r = self.requests[req]
        freed = 0
        if not self._has_window:
            return 0
        for gi, g in enumerate(self.groups):
            w, c = g.need.window, g.need.chunk
            if w is None and c is None:
                continue
            first_needed = 0                                     # lowest key position still visible
            if w is not None:
                first_needed = max(0, r.num_tokens - w + 1)
            if c is not None:
                first_needed = max(first_needed, (r.num_tokens // c) * c)
            first_block = first_needed // self.page_size
            table = r.tables[gi]
            give = []
            for b in range(r.first_live[gi], min(first_block, len(table))):
                if table[b] >= 0:
                    give.append(table[b])
                    table[b] = -1
            if give:
                g.pool.release(give, req)
                freed += len(give)
            r.first_live[gi] = max(r.first_live[gi], min(first_block, len(table)))
        return freed

    def free(self, req: Hashable) -> None:
        r = self.requests.pop(req)
        self.changes += 1
        for g, table in zip(self.groups, r.tables):
            g.pool.release([p for p in table if p >= 0], req)
        self.slots.release(r.state_slot, req)

    def num_free_pages(self) -> List[int]:
        return [g.pool.num_free for g in self.groups]

    def check(self) -> None:
        """No page lost, held twice or free while held; tables agree with the pools."""
        for gi, g in enumerate(self.groups):
            g.pool.check()
            held: Dict[int, List[Hashable]] = {}         # page -> the requests whose tables have it
            for req, r in self.requests.items():
                for p in r.tables[gi]:
                    if p < 0:
                        continue
                    there = held.setdefault(p, [])
                    if there and there[-1] == req:
                        raise SchedulerError(f"page {p} of group {gi} is in the table of {req!r} twice")
                    if there and not (g.pool.holds(p, there[-1]) and g.pool.holds(p, req)):
                        raise SchedulerError(f"page {p} of group {gi} is in the tables of {there[-1]!r} and {req!r}")
                    there.append(req)
                    if not g.pool.holds(p, req):
                        raise SchedulerError(f"page {p} of group {gi}: table of {req!r}, pool says {g.pool.owner(p)!r}")
            for p, there in held.items():
                if g.pool.num_holders(p) != len(there):
                    raise SchedulerError(f"page {p} of group {gi} has {g.pool.num_holders(p)} holders and is in the tables of {there!r}")
            if len(held) + g.pool.num_free != g.pool.num_pages:
                raise SchedulerError(f"group {gi}: {len(held)} held + {g.pool.num_free} free != {g.pool.num_pages}")
        self.slots.check()
