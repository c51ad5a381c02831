"""Which sequences of a step begin with the same cached tokens, and the step's tables as the kernels read them."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from ..errors import KernelError

TILE_ROWS = 128            # rows of a row tile (SP_ROWS of csrc/shared_prefix.cuh)
KEY_TILE = 64              # keys of a tile: ranges of keys begin at multiples of it


def _cut(tiles_of: Sequence[int], kv_heads: int, num_sms: int) -> int:
    """Key tiles of a range: such that the ranges of all row tiles and kv heads are at most one CTA an SM, and no fewer than two where
    that leaves more than six parts to merge (a CTA costs about as much as three tiles to set up and to merge; 3 sequences behind 324
    tokens, 32 heads on 8: 10.7 us in ranges of two tiles, 9.2 of one; 82 behind up to 634, 28 heads on 4: 13.1 and 15.5); where one
    CTA an SM makes them longer than eight, two CTAs an SM (2 to 5 % for prefixes of 8,000 and more; 64 sequences behind 2,048 tokens,
    which have their own keys to read beside, 26.7 us with one and 29.4 with two)."""
    def least(places: int) -> int:
        lo = 1 if max(tiles_of) <= 6 else 2
        hi = max(max(tiles_of), lo)
        while lo < hi:
            mid = (lo + hi) // 2
            if sum(-(-n // mid) for n in tiles_of) * kv_heads <= places:
                hi = mid
            else:
                lo = mid + 1
        return lo
    one = least(num_sms)
    return one if one <= 8 else least(2 * num_sms)


def _staged(host: np.ndarray, device) -> torch.Tensor:
    """The array in memory that a copy to `device` reads without making the host wait for the stream (which as a rule is at work on the
    step before).  Pinned memory from torch's host allocator, which does not hand it out again before the copy has been done."""
    t = torch.from_numpy(host)
    if torch.device(device).type != "cuda":
        return t
    if torch.cuda.is_current_stream_capturing():
        raise KernelError("shared prefixes: groups are laid out and changed outside a capture (a replay would copy memory that is given back)")
    return t.pin_memory()


class SharedPrefixes:
    """The groups of a step's sequences whose first tokens are the same cached ones, laid out for the kernels.

    `groups`: (members, tokens) per group: the places of its sequences in the step and how many leading tokens they share.
    Their block tables must lead to the same keys and values there (as a rule the same pages; the page in which the shared
    tokens end may be a copy).  A sequence belongs to one group at most; groups of one and groups without tokens share nothing
    and are left out.  The object depends on neither the tokens behind the prefixes nor the layer: a program keeps it while
    its set of sequences stays.  It takes part in no computation but `CudaKernels.shared_prefix_attention`.

    `capacity` = (row tiles, ranges of keys): fixes the size of the arrays, so that a captured graph serves other groups of
    the same number of sequences (`refill`).  Without one the launches are sized for the groups given here, and these stay."""

    def __init__(self, groups, num_seqs: int, num_heads: int, num_kv_heads: int, device, capacity: Optional[Tuple[int, int]] = None,
                 num_sms: int = 148):
        if num_seqs < 0 or num_heads < 1 or num_kv_heads < 1 or num_heads % num_kv_heads:
            raise KernelError(f"shared prefixes: {num_seqs} sequences of {num_heads} heads on {num_kv_heads} key/value heads")
        self.num_seqs, self.num_heads, self.num_kv_heads = num_seqs, num_heads, num_kv_heads
        self.num_sms = num_sms
        self.refillable = capacity is not None
        host, (self.num_tiles, self.num_items), sizes = self._lay_out(groups, capacity)
        # with a capacity the launches are sized for any groups that fit it
        self.capacity = capacity or (self.num_tiles, self.num_items)
        if capacity is not None:
            sizes = capacity[1], 0, 1, max(1, TILE_ROWS // (num_heads // num_kv_heads))
        # the most ranges of a row tile, the fewest keys that any sequence has before its own begin (0: one has no prefix), key tiles of
        # a range, sequences of a row tile
        self.most_parts, self.shortest, self.longest, self.widest = sizes
        self._event, self.written_on = None, None
        self.device_ints = _staged(host, device).to(device, non_blocking=True)
        self._note_write()

    def refill(self, groups) -> None:
        """Other groups of the same step size, into the same array (on the current stream).  It takes a capacity given when the object
        was made: otherwise a launch is sized for the first groups (their widest row tile decides how many rows are computed at all)."""
        self.write(self.other(groups))

    def other(self, groups):
        """The array of other groups, as `write` takes it; nothing here changes."""
        if not self.refillable:
            raise KernelError("shared prefixes: laid out for the groups they were made with; other groups need a capacity or a new object")
        return self._lay_out(groups, self.capacity)[:2]

    def write(self, laid_out) -> None:
        host, used = laid_out
        self.device_ints.copy_(_staged(host, self.device_ints.device), non_blocking=True)
        self.num_tiles, self.num_items = used
        self._note_write()

    def _note_write(self) -> None:
        device = self.device_ints.device
        if device.type == "cuda":
            stream = torch.cuda.current_stream(device)
            self._event = self._event or torch.cuda.Event()
            self._event.record(stream)
            self.written_on = stream.cuda_stream

    def wait_for_write(self) -> None:
        """For a call on another stream than the array was written on: the current stream waits for the copy, the host does not.  (A capture
        cannot wait for what is outside it; `torch.cuda.graph` begins one when the device is idle.)"""
        if self._event is not None and not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(self.device_ints.device).wait_event(self._event)

    @staticmethod
    def ints(num_seqs: int, capacity: Tuple[int, int]) -> int:
        """32-bit integers of the array."""
        tiles, items = capacity
        return (4 + 3 * num_seqs + 2 * tiles + 3) // 4 * 4 + 8 * items

    @property
    def own_start(self) -> torch.Tensor:
        """int32 [num_seqs] on the device: the first token of each sequence that lies behind its prefix."""
        return self.device_ints[4:4 + self.num_seqs]

    def _lay_out(self, groups, capacity):
        """(the array, its row tiles and ranges in use, the sizes that a launch for these groups alone goes by)"""
        B, per = self.num_seqs, self.num_heads // self.num_kv_heads
        seen = set()
        kept = []
        for members, tokens in groups:
            members = [int(m) for m in members]
            for m in members:
                if not 0 <= m < B:
                    raise KernelError(f"shared prefixes: sequence {m} of a step of {B}")
                if m in seen:
                    raise KernelError(f"shared prefixes: sequence {m} is in two groups, or twice in one")
                seen.add(m)
            if tokens < 0 or tokens > 0x7fffffff - KEY_TILE:
                raise KernelError(f"shared prefixes: a prefix of {tokens} tokens")
            if len(members) > 1 and tokens > 0:
                kept.append((members, int(tokens)))
        if per > TILE_ROWS and kept:
            raise KernelError(f"shared prefixes: {per} query heads on a key/value head are more than the {TILE_ROWS} rows of a tile")
        tile_members = max(1, TILE_ROWS // per)
        tiles = []                                   # (sequence whose table is read, first member, how many, tokens)
        flat, own_start, place = [], np.zeros(B, np.int32), np.full(B, -1, np.int32)
        for members, tokens in kept:
            for at in range(0, len(members), tile_members):
                part = members[at:at + tile_members]
                for i, m in enumerate(part):
                    own_start[m] = tokens
                    place[m] = len(tiles) * TILE_ROWS + i * per
                tiles.append((members[0], len(flat), len(part), tokens))
                flat.extend(part)
        key_tiles = [-(-t[3] // KEY_TILE) for t in tiles]
        items, parts = [], []
        if tiles:
            step = _cut(key_tiles, self.num_kv_heads, self.num_sms)
            for i, n in enumerate(key_tiles):
                k = -(-n // step)
                edges = [n * j // k for j in range(k + 1)]
                parts.append((len(items), k))
                seq, first, count, tokens = tiles[i]
                items += [(a * KEY_TILE, min(b * KEY_TILE, tokens), seq, first, count, i, 0, 0) for a, b in zip(edges, edges[1:])]
        capacity = capacity or (len(tiles), len(items))
        if len(tiles) > capacity[0] or len(items) > capacity[1]:
            raise KernelError(f"shared prefixes: {len(tiles)} row tiles and {len(items)} ranges of keys do not fit a capacity of {capacity}")
        host = np.zeros(self.ints(B, capacity), np.int32)
        host[0], host[1] = len(items), len(tiles)
        host[4:4 + B] = own_start
        host[4 + B:4 + 2 * B] = place
        host[4 + 2 * B:4 + 2 * B + len(flat)] = flat
        if tiles:
            host[4 + 3 * B:4 + 3 * B + 2 * len(tiles)] = np.asarray(parts, np.int32).ravel()
            at = (4 + 3 * B + 2 * capacity[0] + 3) // 4 * 4
            host[at:at + 8 * len(items)] = np.asarray(items, np.int32).ravel()
        sizes = (max((n for _, n in parts), default=0), min((t for _, t in kept), default=0) if len(flat) == B else 0,
                 step if tiles else 0, max((t[2] for t in tiles), default=0))
        return host, (len(tiles), len(items)), sizes


class StepPrefixes:
    """The groups of a step for every layout of heads that its layers have (one `SharedPrefixes` each, made when a layer first asks).

    `most_groups`: fixes the arrays' capacities for up to so many groups; `set_groups` then fills them anew, wherever a captured
    graph holds them."""

    def __init__(self, groups, num_seqs: int, device, most_groups: Optional[int] = None, num_sms: int = 148):
        self.groups = self._own(groups)
        self.num_seqs, self.device, self.most_groups, self.num_sms = num_seqs, device, most_groups, num_sms
        self._layouts = {}

    @property
    def used(self) -> bool:
        """Whether any layer has asked for a layout."""
        return bool(self._layouts)

    @staticmethod
    def _own(groups):
        """A copy: the caller may go on with its lists."""
        return [(list(members), tokens) for members, tokens in groups]

    def layout(self, num_heads: int, num_kv_heads: int) -> SharedPrefixes:
        made = self._layouts.get((num_heads, num_kv_heads))
        if made is None:
            capacity = None
            if self.most_groups is not None:
                members = max(1, TILE_ROWS // (num_heads // num_kv_heads))
                tiles = -(-self.num_seqs // members) + self.most_groups
                capacity = (tiles, tiles + -(-2 * self.num_sms // num_kv_heads))
            made = SharedPrefixes(self.groups, self.num_seqs, num_heads, num_kv_heads, self.device, capacity, self.num_sms)
            self._layouts[(num_heads, num_kv_heads)] = made
        return made

    def set_groups(self, groups) -> None:
        groups = self._own(groups)
        if groups == self.groups:
            return
        if self.most_groups is None or len(groups) > self.most_groups:
            raise KernelError(f"shared prefixes: {len(groups)} groups where {self.most_groups} fit")
        # all layouts first: groups that one of them refuses leave the arrays, and what this object takes them to hold, as they were
        laid_out = [(made, made.other(groups)) for made in self._layouts.values()]
        for made, host in laid_out:
            made.write(host)
        self.groups = groups


@dataclass(slots=True)
class StepTables:
    """What `CudaKernels.step_tables` writes (int32, on the device)."""
    block_tables: torch.Tensor         # [groups, sequences, max_blocks]
    slot_mapping: torch.Tensor         # [groups, tokens]
    positions: torch.Tensor            # [tokens]
    token_seq: torch.Tensor            # [tokens]
    cu_seqlens: torch.Tensor           # [sequences + 1]
    ctx_lens: torch.Tensor             # [sequences]
