"""The step function: one batch of (request, its next tokens) through the model.

A batch holds, in any order, whole prompts, portions of prompts cut anywhere and single
decoded tokens.  The step reserves cache room for exactly the tokens it is given, packs the
batch's metadata into one pinned buffer that goes to the device in one copy, runs the model
over these tokens against the cache that earlier steps left, and returns float32 logits at
the wanted places.

The reference runs a step either as all-decode or as all-prefill of equal-length prompts
(v3/crates/rvllm-runtime/src/layer_exec.rs:32-39,367-372; scheduler.rs:1-6) and fills its
metadata with separate synchronous copies (bring_up.rs:698-708); its packed layout
(v3/crates/rvllm-metadata/src/layout.rs:19-55: token ids, positions, context lengths, block
tables, slot mapping, sequence starts; padding rows have slot -1, pack.rs:79-86) is what the
buffer here follows, extended per cache group.

Where the kernel library offers `step_tables`, the buffer holds the requests' lengths and the pages handed out since the last
step, and the block tables, slot maps, positions and sequence starts are built on the device, in front of a table of all
requests' pages that stays there; otherwise the host writes them out.
"""
from __future__ import annotations

import gc
from dataclasses import dataclass, field
from typing import Dict, Hashable, List, Optional, Sequence

import numpy as np
import torch

from ..cache import CacheManager
from ..errors import KvExhausted, SchedulerError
from ..kernels.library import COUNTERS, AttentionMeta
from ..kernels.shared import StepPrefixes, StepTables

SHARED_MOST_GROUPS = 8         # groups of a captured step: those that save the most
# A decode step reads shared beginnings once, instead of as many times as requests hold them, where that is the faster way:
# * bfloat16: the keys and values it saves a layer are this many bytes and half of those that it reads sequence by sequence.  32 heads of
#   128 on 8, each for itself and shared, us: 16 requests with 16 keys of their own behind 256 (15.7 MB saved) 9.1 and 8.7, behind
#   512 10.5 and 9.4, 8 behind 2,048 (59 MB) 13.3 and 11.1, 64 with 1,024 of their own (268 MB) behind 512 (132 MB) 59 and 54,
#   behind 2,048 94 and 59, with 16 behind 8,192 226 and 26;
SHARED_MIN_BYTES = 24 << 20
#   ... and twice as many in a graph, which is launched for any groups that fit it (1 to 4 us a layer that a layout of the very groups does
#   without), unless it has this many (sequence, kv head) pairs, where reading each for itself costs more, or one kv head, where it has
#   few CTAs.  Each for itself and shared in a graph, us: 16 behind 512 10.4 and 11.0, 2 behind 8,192 (34 MB) 15.5 and 17.7, with 800 of
#   their own 16.1 and 21.5; 64 behind 128 (33 MB) 16.4 and 12.3, 28 heads on 4 64 behind 256 (33 MB) 18.0 and 12.7, 16 on one
#   32 behind 2,048 (33 MB) 16.5 and 12.0.  (336 sizes of 8 to 170 MB saved, six layouts of heads: 1.7 % above the
#   better of the two in all, 8 % above each for itself at worst; with the one threshold 3.4 and 34 %.)
SHARED_GRAPH_MIN_BYTES = 48 << 20
SHARED_GRAPH_MANY_PAIRS = 256
# * float32: some beginning is this long (28 heads of 128 on 4: 4 requests with 16 keys of their own behind 64 8.3 and 12.5 us, behind
#   256 17.0 and 12.9, 16 behind 1,024 105 and 31; in a graph 15.7, 17.1 and 33), or the bytes saved are half of the above (64 behind
#   64: 46 and 15.4, in a graph 18.8).  What it does not ask for is the heads on a kv head: with one, own keys take longer shared than each
#   for itself (16 heads of 64 on 16, 64 requests with 800 of their own behind 512 241 and 257).
SHARED_MIN_TOKENS_F32 = 256


@dataclass
class StepEntry:
    """One request's share of a step: its next tokens and the places (indices into `tokens`)
    whose logits are wanted."""
    req_id: Hashable
    tokens: Sequence[int]
    want: Sequence[int] = ()


class StepContext:
    """What the parts see of a step."""
    __slots__ = ("kernels", "num_tokens", "num_seqs", "token_ids", "positions", "token_seq", "cu_seqlens",
                 "state_slots", "logit_rows", "attention", "q_lens", "ctx_lens", "req_ids", "extras", "following_norms")

    def __init__(self):
        self.extras = {}
        self.following_norms = None      # the norms in front of the block that runs next, if this block may form them (parts/base.py)


class ModelRunner:
    def __init__(self, model, cache: CacheManager, kernels, max_model_len: int, device,
                 graph_batch_sizes: Sequence[int] = ()):
        self.model, self.cache, self.kernels = model, cache, kernels
        self.graph_batch_sizes = tuple(sorted(graph_batch_sizes))
        self._graphs = {}
        self._graph_pool = None
        self._graph_event = None
        self.max_model_len = max_model_len
        self.device = torch.device(device)
        self.max_blocks = cache.blocks_for(max_model_len)
        # a small ring of pinned staging buffers: a buffer is rewritten only after the copy that
        # last read it has finished, so the host never waits for the step it has just launched
        self._ring: List[Optional[torch.Tensor]] = [None, None, None]
        self._ring_events: List[Optional[object]] = [None, None, None]
        self._ring_next = 0
        self._dev: Optional[torch.Tensor] = None
        # the requests of the last decode step (and how often the cache's had changed), which of them share beginnings, and the layout
        # that eager steps have for these groups
        self._groups_of = (None, [])
        self._eager_prefixes: Optional[StepPrefixes] = None
        # bytes of a key and its value in the largest of the groups whose shared beginnings are read once (0: there is no such group)
        needs = [g.need for g in cache.groups if self._reads_once(g.need)]
        widest = max(needs, key=lambda n: n.num_kv_heads * n.row_elements, default=None)
        self._kv_heads = widest.num_kv_heads if widest else 0
        self._key_bytes = self._kv_heads * widest.row_elements * torch.empty((), dtype=cache.dtype).element_size() if widest else 0
        self._least_saved = SHARED_MIN_BYTES
        self._page_table = None
        if cache.groups and self.device.type == "cuda" and hasattr(kernels, "step_tables"):
            G = len(cache.groups)
            self._page_table = torch.full((G, cache.max_seqs, self.max_blocks), -1, dtype=torch.int32, device=self.device)
            self._spans = torch.tensor([[g.need.window or 0, g.need.chunk or 0] for g in cache.groups], dtype=torch.int32, device=self.device)
        self.steps_run = 0
        self.last_h2d_bytes = 0

    # ---- metadata buffers --------------------------------------------------------------------
    def _buffers(self, n_ints: int):
        i = self._ring_next
        self._ring_next = (i + 1) % len(self._ring)
        if self._ring_events[i] is not None:
            self._ring_events[i].synchronize()
        size = max(n_ints, 1 << 16)
        if self._ring[i] is None or self._ring[i].numel() < n_ints:
            self._ring[i] = torch.empty((size,), dtype=torch.int32, pin_memory=self.device.type == "cuda")
        if self._dev is None or self._dev.numel() < n_ints:
            self._dev = torch.empty((size,), dtype=torch.int32, device=self.device)
        return i, self._ring[i], self._dev

    # ---- one step ----------------------------------------------------------------------------
    def validate(self, entries: Sequence[StepEntry]) -> None:
        vocab = self.model.spec.vocab_size
        seen = set()
        for e in entries:
            if e.req_id in seen:
                raise SchedulerError(f"request {e.req_id!r} appears twice in one step")
            seen.add(e.req_id)
            n_tok = len(e.tokens)
            if n_tok == 0:
                raise SchedulerError(f"request {e.req_id!r} brings no tokens to the step")
            if n_tok == 1:
                bad = [] if 0 <= e.tokens[0] < vocab else [e.tokens[0]]
            else:
                lo, hi = min(e.tokens), max(e.tokens)
                bad = [] if (0 <= lo and hi < vocab) else [t for t in e.tokens if not 0 <= int(t) < vocab]
            if bad:
                raise SchedulerError(f"request {e.req_id!r}: token id {bad[0]} is outside the vocabulary of {vocab}")
            have = self.cache.num_tokens(e.req_id) if self.cache.has(e.req_id) else 0
            if have + len(e.tokens) > self.max_model_len:
                raise SchedulerError(f"request {e.req_id!r}: {have} + {len(e.tokens)} tokens exceed max_model_len {self.max_model_len}")
            for w in e.want:
                if not 0 <= w < len(e.tokens):
                    raise SchedulerError(f"request {e.req_id!r}: wanted place {w} is outside its {len(e.tokens)} tokens")

    def reserve(self, entries: Sequence[StepEntry]) -> List[int]:
        """Admit unknown requests and take the pages of the whole batch, or nothing."""
        cache = self.cache
        n_groups = len(cache.groups)
        total = [0] * n_groups
        new = 0
        for e in entries:
            known = cache.has(e.req_id)
            new += 0 if known else 1
            need = cache.pages_needed(e.req_id if known else None, len(e.tokens))
            for g in range(n_groups):
                total[g] += need[g]
        if any(total):
            for need, have in zip(total, cache.num_free_pages()):
                if need > have:
                    raise KvExhausted(need, have, "the step's tokens do not fit the free pages")
        if new > cache.slots.num_free:
            raise SchedulerError(f"{new} new requests but only {cache.slots.num_free} request slots are free")
        starts = []
        for e in entries:
            if not cache.has(e.req_id):
                cache.admit(e.req_id)
            starts.append(cache.append(e.req_id, len(e.tokens)))
        return starts

    def pack(self, entries: Sequence[StepEntry], starts: List[int], pad_to: Optional[int] = None,
             buffers=None, late=None, ctx_limit: Optional[int] = None) -> StepContext:
        """Write the step's metadata into a pinned buffer and send it to the device in one copy.

        With `pad_to` the batch is padded to that many one-token sequences (padding rows: token
        0, context length 0, slot -1, state slot -1 - they write nothing and attend to nothing;
        v3/crates/rvllm-metadata/src/pack.rs:35-40,79-86 of the reference pads the same way), block
        tables get the full width, and the layout depends on `pad_to` alone, so that a captured
        CUDA graph can be replayed on the buffer; `ctx_limit` is then the context length that the
        graph's kernels are laid out for (no sequence of the batch is longer).

        `late` = (sampled ids on the device, one index per entry): an entry with index j >= 0 is a
        one-token sequence whose token is sampled[j], which the host has not read; its token is
        put in place on the device after the copy."""
        if self._page_table is not None:
            return self._pack_lengths(entries, starts, pad_to, buffers, late, ctx_limit)
        cache = self.cache
        n_real = len(entries)
        B = pad_to if pad_to is not None else n_real
        q_lens = [len(e.tokens) for e in entries] + [1] * (B - n_real)
        T = sum(q_lens)
        ctx_lens = [s + n for s, n in zip(starts, q_lens)] + [0] * (B - n_real)
        wants = [list(e.want) for e in entries]
        if pad_to is not None:
            wants = [[0]] * B
        R = sum(len(w) for w in wants)
        G = len(cache.groups)
        MB = self.max_blocks if pad_to is not None else max(1, cache.blocks_for(max(ctx_lens)))
        n_ints = 3 * T + (B + 1) + 2 * B + R + G * (T + B * MB) + B + 16
        if buffers is None:
            ring_i, host, dev = self._buffers(n_ints)
        else:
            ring_i, (host, dev) = None, buffers
        h = host.numpy()
        off = 0

        def take(n):
            nonlocal off
            a = off
            off += n
            return a

        o_tok, o_pos, o_seq = take(T), take(T), take(T)
        o_cu, o_ctx, o_state, o_rows = take(B + 1), take(B), take(B), take(R)
        if pad_to is not None:
            return self._pack_decode(entries, starts, B, MB, h, host, dev,
                                     (o_tok, o_pos, o_seq, o_cu, o_ctx, o_state, o_rows), take, late,
                                     ctx_limit or self.max_model_len)
        cu = 0
        rows: List[int] = []
        h[o_cu] = 0
        for i in range(B):
            n = q_lens[i]
            if i < n_real:
                e = entries[i]
                h[o_tok + cu:o_tok + cu + n] = np.asarray(e.tokens, dtype=np.int32)
                h[o_pos + cu:o_pos + cu + n] = np.arange(starts[i], starts[i] + n, dtype=np.int32)
                h[o_state + i] = cache.state_slot(e.req_id)
            else:
                h[o_tok + cu] = 0
                h[o_pos + cu] = 0
                h[o_state + i] = -1
            h[o_seq + cu:o_seq + cu + n] = i
            rows.extend(cu + w for w in wants[i])
            cu += n
            h[o_cu + i + 1] = cu
            h[o_ctx + i] = ctx_lens[i]
        if R:
            h[o_rows:o_rows + R] = np.asarray(rows, dtype=np.int32)
        group_offsets = []
        ps = cache.page_size
        for gi in range(G):
            o_slot, o_bt = take(T), take(B * MB)
            h[o_bt:o_bt + B * MB] = -1
            h[o_slot:o_slot + T] = -1
            cu = 0
            for i, e in enumerate(entries):
                table = cache.block_table(e.req_id, gi)
                nb = len(table)
                tb = np.asarray(table, dtype=np.int32)
                h[o_bt + i * MB:o_bt + i * MB + nb] = tb
                pos = np.arange(starts[i], starts[i] + q_lens[i])
                h[o_slot + cu:o_slot + cu + q_lens[i]] = tb[pos // ps] * ps + pos % ps
                cu += q_lens[i]
            group_offsets.append((o_slot, o_bt))
        o_late = take(B)
        if late is not None:
            h[o_late:o_late + n_real] = late[1]
            h[o_late + n_real:o_late + B] = -1
        dev[:off].copy_(host[:off], non_blocking=True)
        self.last_h2d_bytes = off * 4
        if self.device.type == "cuda" and ring_i is not None:
            ev = self._ring_events[ring_i] or torch.cuda.Event()
            ev.record()
            self._ring_events[ring_i] = ev

        ctx = StepContext()
        ctx.kernels = self.kernels
        ctx.num_tokens, ctx.num_seqs = T, B
        ctx.token_ids = dev[o_tok:o_tok + T]
        ctx.positions = dev[o_pos:o_pos + T]
        ctx.token_seq = dev[o_seq:o_seq + T]
        ctx.cu_seqlens = dev[o_cu:o_cu + B + 1]
        if late is not None:
            self.kernels.late_tokens(ctx.token_ids, ctx.cu_seqlens, dev[o_late:o_late + B], late[0])
        dev_ctx = dev[o_ctx:o_ctx + B]
        ctx.state_slots = dev[o_state:o_state + B]
        ctx.logit_rows = dev[o_rows:o_rows + R]
        ctx.q_lens, ctx.ctx_lens = q_lens, ctx_lens
        ctx.req_ids = [e.req_id for e in entries]
        ctx.attention = []
        max_ctx = self.max_model_len if pad_to is not None else max(ctx_lens)
        for (o_slot, o_bt) in group_offsets:
            ctx.attention.append(AttentionMeta(
                block_tables=dev[o_bt:o_bt + B * MB].view(B, MB), cu_seqlens=ctx.cu_seqlens, ctx_lens=dev_ctx,
                token_seq=ctx.token_seq, slot_mapping=dev[o_slot:o_slot + T], num_seqs=B,
                max_q_len=max(q_lens), max_ctx_len=max_ctx, page_size=ps,
                num_decode=sum(1 for n in q_lens if n == 1)))
        return ctx

    def _new_pages(self, entries) -> int:
        """Pages of the entries that the table on the device does not have yet."""
        return sum(len(t) - n for e in entries for r in (self.cache.requests[e.req_id],) for t, n in zip(r.tables, r.on_device))

    def _pack_lengths(self, entries, starts, pad_to, buffers, late, ctx_limit) -> StepContext:
        """`pack` where the device builds the tables: the buffer holds, in this order, state slots, starts and token counts of the
        sequences, the blocks that each has on the device by group, tokens, wanted rows, sources of late tokens, new pages; behind
        them (on the device only) lie the tables that are built."""
        cache = self.cache
        n_real, G = len(entries), len(cache.groups)
        B = pad_to if pad_to is not None else n_real
        pads = B - n_real
        q_lens = [len(e.tokens) for e in entries] + [1] * pads
        T = sum(q_lens)
        ctx_lens = [s + n for s, n in zip(starts, q_lens)] + [0] * pads
        held = [cache.requests[e.req_id] for e in entries]
        if pad_to is not None:
            rows = np.arange(B, dtype=np.int32)
            MB, room = self.max_blocks, G * B                      # (a decoded token takes one page of a group at most)
        else:
            ends = np.cumsum([0] + q_lens)
            rows = np.asarray([ends[i] + w for i, e in enumerate(entries) for w in e.want], dtype=np.int32)
            MB, room = max(1, cache.blocks_for(max(ctx_lens))), self._new_pages(entries)
        R = len(rows)
        sent = 3 * B + G * B + T + R + B + max(room, 1)
        built = (G * B * MB, G * T, T, T, B + 1, B)
        if buffers is None:
            ring_i, host, dev = self._buffers(sent + sum(built))
        else:
            ring_i, (host, dev) = None, buffers
        h = host.numpy()
        o_start, o_q, o_held = B, 2 * B, 3 * B
        o_tok = o_held + G * B
        o_rows, o_late, o_new = o_tok + T, o_tok + T + R, o_tok + T + R + B
        h[:n_real] = [r.state_slot for r in held]
        h[n_real:B] = -1
        h[o_start:o_start + n_real] = starts
        h[o_start + n_real:o_start + B] = 0
        h[o_q:o_q + B] = q_lens
        h[o_rows:o_rows + R] = rows
        if T == B:
            h[o_tok:o_tok + n_real] = [e.tokens[0] for e in entries]
            h[o_tok + n_real:o_tok + T] = 0
        else:
            at = o_tok
            for e, n in zip(entries, q_lens):
                h[at:at + n] = e.tokens
                at += n
        at = o_new
        for g in range(G):
            h[o_held + g * B:o_held + g * B + n_real] = [r.on_device[g] for r in held]
            h[o_held + g * B + n_real:o_held + (g + 1) * B] = 0
            for r in held:
                new = r.tables[g][r.on_device[g]:]
                if new:
                    h[at:at + len(new)] = new
                    at += len(new)
        h[o_late:o_late + n_real] = late[1] if late is not None else -1
        h[o_late + n_real:o_late + B] = -1
        dev[:at].copy_(host[:at], non_blocking=True)
        self.last_h2d_bytes = at * 4
        if ring_i is not None:
            ev = self._ring_events[ring_i] or torch.cuda.Event()
            ev.record()
            self._ring_events[ring_i] = ev

        tables, slots, positions, token_seq, cu, ctx_dev = dev[sent:sent + sum(built)].split_with_sizes(built)
        made = StepTables(tables.view(G, B, MB), slots.view(G, T), positions, token_seq, cu, ctx_dev)
        self.kernels.step_tables(self._page_table, dev[:B], dev[o_held:o_tok].view(G, B), dev[o_start:o_q], dev[o_q:o_held], dev[o_new:max(at, o_new + 1)],
                                 self._spans, T, MB, cache.page_size, out=made,
                                 settle=late is None and (pad_to is None or not entries))    # (otherwise `late_tokens` or a graph is next)
        for r in held:
            r.on_device = [len(t) for t in r.tables]
        ctx = StepContext()
        ctx.kernels = self.kernels
        ctx.num_tokens, ctx.num_seqs = T, B
        ctx.token_ids = dev[o_tok:o_tok + T]
        ctx.positions, ctx.token_seq, ctx.cu_seqlens = positions, token_seq, cu
        if late is not None:
            self.kernels.late_tokens(ctx.token_ids, cu, dev[o_late:o_late + B], late[0])
        ctx.state_slots = dev[:B]
        ctx.logit_rows = dev[o_rows:o_rows + R]
        ctx.q_lens, ctx.ctx_lens = q_lens, ctx_lens
        ctx.req_ids = [e.req_id for e in entries]
        longest = (ctx_limit or self.max_model_len) if pad_to is not None else max(ctx_lens)
        ctx.attention = [AttentionMeta(block_tables=made.block_tables[g], cu_seqlens=cu, ctx_lens=ctx_dev, token_seq=token_seq,
                                       slot_mapping=made.slot_mapping[g], num_seqs=B, max_q_len=max(q_lens), max_ctx_len=longest,
                                       page_size=cache.page_size, num_decode=q_lens.count(1)) for g in range(G)]
        return ctx

    # ---- beginnings that requests share ----------------------------------------------------------
    def _reads_once(self, need) -> bool:
        """Whether the attention of a cache group may read beginnings that sequences share once (one row for key and value, values of
        another size than keys and windows have kernels of their own, which read each sequence for itself)."""
        if need.planes != 2 or need.flat_pages or need.window is not None or need.chunk is not None:
            return False
        rule = getattr(self.kernels, "reads_prefixes_once", None)
        return rule is not None and rule(self.cache.dtype, need.num_kv_heads, need.head_dim, self.cache.page_size, self.cache.num_pages, self.cache.max_seqs)

    def _shared_groups(self, entries, starts, graph: bool = False):
        """(places, tokens) per group of entries that begin with the same cached tokens, for a step of decoded tokens (`graph`: one that
        runs from a captured graph); none where it would not pay.  Pages that are shared stay as they are while their requests live, so the groups hold until the set of
        requests changes."""
        if not self._key_bytes or not self.cache.any_shared or self._page_table is None or any(len(e.tokens) != 1 for e in entries):
            return []
        reqs = (self.cache.changes, tuple(e.req_id for e in entries))
        if reqs != self._groups_of[0]:
            groups = sorted(self.cache.shared_groups(reqs[1]), key=lambda g: -(len(g[0]) - 1) * g[1])
            self._groups_of = (reqs, groups)
        groups = self._groups_of[1][:SHARED_MOST_GROUPS] if graph else self._groups_of[1]
        self._least_saved = self._graph_least(len(entries)) if graph else SHARED_MIN_BYTES
        return groups if groups and self._worth_sharing(groups, sum(starts) + len(starts)) else []

    def _worth_sharing(self, groups, keys: int) -> bool:
        """Whether a step of `keys` keys in all takes less time with the groups' beginnings read once (the figures are at the top)."""
        saved = sum((len(m) - 1) * t for m, t in groups)
        own = keys - sum(len(m) * t for m, t in groups)
        if self.cache.dtype == torch.float32:
            return max(t for _, t in groups) >= SHARED_MIN_TOKENS_F32 or saved * self._key_bytes >= SHARED_MIN_BYTES // 2
        return saved * self._key_bytes >= getattr(self, "_least_saved", SHARED_MIN_BYTES) + own * self._key_bytes // 2

    def _may_share(self, num_seqs: int, context: int) -> bool:
        """Whether a graph of so many sequences in contexts up to `context` ever reads shared beginnings once: in a step of all of them that
        differ in their last tokens only."""
        if not self._key_bytes or not self.cache.can_share or self._page_table is None or num_seqs < 2:
            return False
        self._least_saved = self._graph_least(num_seqs)
        return self._worth_sharing([(list(range(num_seqs)), context - 1)], num_seqs * context)

    def _graph_least(self, num_seqs: int) -> int:
        few = 1 < self._kv_heads and num_seqs * self._kv_heads < SHARED_GRAPH_MANY_PAIRS
        return SHARED_GRAPH_MIN_BYTES if few else SHARED_MIN_BYTES

    def _eager_shared(self, groups, num_seqs: int) -> StepPrefixes:
        last = self._eager_prefixes
        if last is None or last.num_seqs != num_seqs or last.groups != groups:
            last = self._eager_prefixes = StepPrefixes(groups, num_seqs, self.device, num_sms=self.kernels.num_sms)
        return last

    @staticmethod
    def _longest_own(starts, groups) -> int:
        """The most keys that an entry has behind its group's beginning, this step's token included."""
        own = [s + 1 for s in starts]
        for members, tokens in groups:
            for m in members:
                own[m] -= tokens
        return max(own)

    def _pack_decode(self, entries, starts, B, MB, h, host, dev, offs, take, late=None, ctx_limit=None) -> StepContext:
        """`pack` for a padded batch of one-token sequences (T = R = B): whole-array writes."""
        cache = self.cache
        o_tok, o_pos, o_seq, o_cu, o_ctx, o_state, o_rows = offs
        n = len(entries)
        ar = np.arange(B + 1, dtype=np.int32)
        h[o_tok:o_tok + B] = 0
        h[o_pos:o_pos + B] = 0
        h[o_ctx:o_ctx + B] = 0
        h[o_state:o_state + B] = -1
        if n:
            h[o_tok:o_tok + n] = [e.tokens[0] for e in entries]
            h[o_pos:o_pos + n] = starts
            h[o_ctx:o_ctx + n] = np.asarray(starts, dtype=np.int32) + 1
            h[o_state:o_state + n] = [cache.state_slot(e.req_id) for e in entries]
        h[o_seq:o_seq + B] = ar[:B]
        h[o_cu:o_cu + B + 1] = ar
        h[o_rows:o_rows + B] = ar[:B]
        ps = cache.page_size
        group_offsets = []
        for gi in range(len(cache.groups)):
            o_slot, o_bt = take(B), take(B * MB)
            bt = h[o_bt:o_bt + B * MB].reshape(B, MB)
            bt[:] = -1
            h[o_slot:o_slot + B] = -1
            for i, e in enumerate(entries):
                table = cache.block_table(e.req_id, gi)
                bt[i, :len(table)] = table
                pos = starts[i]
                h[o_slot + i] = table[pos // ps] * ps + pos % ps
            group_offsets.append((o_slot, o_bt))
        o_late = take(B)
        off = o_late
        if late is not None:
            h[o_late:o_late + n] = late[1]
            h[o_late + n:o_late + B] = -1
            off = o_late + B
        dev[:off].copy_(host[:off], non_blocking=True)
        self.last_h2d_bytes = off * 4
        ctx = StepContext()
        ctx.kernels = self.kernels
        ctx.num_tokens, ctx.num_seqs = B, B
        ctx.token_ids = dev[o_tok:o_tok + B]
        ctx.positions = dev[o_pos:o_pos + B]
        ctx.token_seq = dev[o_seq:o_seq + B]
        ctx.cu_seqlens = dev[o_cu:o_cu + B + 1]
        if late is not None:
            self.kernels.late_tokens(ctx.token_ids, ctx.cu_seqlens, dev[o_late:o_late + B], late[0])
        dev_ctx = dev[o_ctx:o_ctx + B]
        ctx.state_slots = dev[o_state:o_state + B]
        ctx.logit_rows = dev[o_rows:o_rows + B]
        ctx.q_lens = [1] * B
        ctx.ctx_lens = [s + 1 for s in starts] + [0] * (B - n)
        ctx.req_ids = [e.req_id for e in entries]
        ctx.attention = [AttentionMeta(
            block_tables=dev[o_bt:o_bt + B * MB].view(B, MB), cu_seqlens=ctx.cu_seqlens, ctx_lens=dev_ctx,
            token_seq=ctx.token_seq, slot_mapping=dev[o_slot:o_slot + B], num_seqs=B, max_q_len=1,
            max_ctx_len=ctx_limit or self.max_model_len, page_size=ps, num_decode=B) for (o_slot, o_bt) in group_offsets]
        return ctx

    def _apply_launch_mode(self) -> None:
        """Tell the kernel library, which the engines of a process share, how this model's kernels follow one another."""
        set_pdl = getattr(self.kernels, "set_pdl", None)
        if set_pdl is not None:
            set_pdl(getattr(getattr(self.model, "spec", None), "programmatic_launch", True))

    def step(self, entries: Sequence[StepEntry], late_tokens=None) -> Optional[torch.Tensor]:
        """Run the batch.  Returns float32 logits [wanted places, vocab] in the order of the
        entries and of each entry's `want` (None if nothing is wanted).

        `late_tokens` = (ids, index): ids is an int32 tensor on the device (what the previous step
        sampled), index has one number per entry; an entry with index j >= 0 brings one token whose
        value is ids[j] and is not known on the host yet (its `tokens` holds a stand-in)."""
        if not entries:
            return None
        self.validate(entries)
        self._apply_launch_mode()
        if late_tokens is not None:
            if len(late_tokens[1]) != len(entries):
                raise SchedulerError(f"{len(entries)} entries but {len(late_tokens[1])} late-token indices")
            for e, j in zip(entries, late_tokens[1]):
                if j >= 0 and len(e.tokens) != 1:
                    raise SchedulerError(f"request {e.req_id!r}: a late token stands for exactly one token")
            if all(j < 0 for j in late_tokens[1]):
                late_tokens = None
        starts = self.reserve(entries)
        bucket = self._graph_bucket(entries)
        if bucket is not None:
            logits = self._step_graph(entries, starts, bucket, late_tokens)
        else:
            ctx = self.pack(entries, starts, late=late_tokens)
            groups = self._shared_groups(entries, starts)
            if groups:
                shared = self._eager_shared(groups, len(entries))
                for m in ctx.attention:
                    m.shared, m.max_own_len = shared, self._longest_own(starts, groups)
            hidden = self.model.forward(ctx, self.cache)
            logits = self.model.compute_logits(hidden, ctx) if ctx.logit_rows.numel() else None
            if groups and not shared.used:
                self._key_bytes = 0
        for e in entries:
            self.cache.release_passed(e.req_id)
        self.steps_run += 1
        return logits

    # ---- decode steps replayed from CUDA graphs -------------------------------------------------
    def _graph_bucket(self, entries: Sequence[StepEntry]) -> Optional[int]:
        """The batch-size bucket whose graph can run this step: every entry brings one token and
        wants its logits, and a bucket is large enough."""
        if not self.graph_batch_sizes or self.device.type != "cuda":
            return None
        if not getattr(self.model, "graph_safe", True):
            return None                       # a part of this model cannot be captured: every step runs eagerly
        for e in entries:
            if len(e.tokens) != 1 or len(e.want) != 1:
                return None
        for b in self.graph_batch_sizes:
            if b >= len(entries):
                return b
        return None

    def _ctx_bucket(self, longest: int) -> int:
        """The context length a graph is laid out for: 512, 768, 1024, 1536, 2048, ... (the attention
        kernel's split of the keys depends on it), at most max_model_len."""
        b = 512
        while b < longest:
            b = b * 3 // 2 if (b & (b - 1)) == 0 else b // 3 * 4
        return min(b, self.max_model_len)

    def _step_graph(self, entries, starts, bucket: int, late=None) -> torch.Tensor:
        ctx_limit = self._ctx_bucket(max(starts) + 1)
        groups = self._shared_groups(entries, starts, graph=True)
        # a step that reads shared beginnings once is another graph, laid out for the keys behind them
        own_limit = self._ctx_bucket(self._longest_own(starts, groups)) if groups else 0
        bucket = (bucket, ctx_limit, own_limit)
        state = self._graphs.get(bucket)
        if state is None or (self._page_table is not None and self._new_pages(entries) > len(self.cache.groups) * len(entries)):
            # the first step of a bucket runs eagerly: it loads every kernel library and lets the
            # GEMM library set itself up; the graph is captured right after it for later steps
            # (so does one whose requests have just taken over pages that the device's table lacks)
            ctx = self.pack(entries, starts, late=late)
            if groups:
                shared = self._eager_shared(groups, len(entries))
                for m in ctx.attention:
                    m.shared, m.max_own_len = shared, own_limit
            hidden = self.model.forward(ctx, self.cache)
            logits = self.model.compute_logits(hidden, ctx)
            if groups and not shared.used:
                self._key_bytes = 0            # no layer reads beginnings once (their attention is another): no graphs of such steps
            elif state is None:
                self._graphs[bucket] = self._capture(*bucket)
            return logits
        host, dev, graph, out, launches, shared = state
        self._graph_event.synchronize()
        self.pack(entries, starts, pad_to=bucket[0], buffers=(host, dev), late=late, ctx_limit=ctx_limit)
        if shared is not None:
            shared.set_groups(groups)
        self._graph_event.record()
        graph.replay()
        COUNTERS["launches"] += launches       # the kernels of this project inside the replayed graph
        return out[:len(entries)]

    def _graph_buffers(self, bucket: int):
        """Staging and device buffer of a captured step of `bucket` sequences, in either form of `pack`."""
        G = len(self.cache.groups)
        n_ints = 8 * bucket + 2 + 2 * G * bucket + G * (bucket + bucket * self.max_blocks) + 5 * bucket + 16
        return torch.empty((n_ints,), dtype=torch.int32, pin_memory=True), torch.empty((n_ints,), dtype=torch.int32, device=self.device)

    def _capture(self, bucket: int, ctx_limit: int, own_limit: int = 0):
        host, dev = self._graph_buffers(bucket)
        ctx = self.pack([], [], pad_to=bucket, buffers=(host, dev), ctx_limit=ctx_limit)   # all rows padded: writes nothing
        shared = None
        if own_limit:
            shared = StepPrefixes([], bucket, self.device, SHARED_MOST_GROUPS, self.kernels.num_sms)
            for m in ctx.attention:
                m.shared, m.max_own_len = shared, own_limit
            self.model.compute_logits(self.model.forward(ctx, self.cache), ctx)     # (makes the layouts, which no capture may)
        torch.cuda.synchronize(self.device)
        graph = torch.cuda.CUDAGraph()
        before = COUNTERS["launches"]
        # no garbage collection meanwhile: it may be that of an engine with graphs of its own, and destroying these ends the capture
        collects = gc.isenabled()
        gc.disable()
        try:
            with torch.cuda.graph(graph, pool=self._graph_pool):
                hidden = self.model.forward(ctx, self.cache)
                out = self.model.compute_logits(hidden, ctx)
        finally:
            if collects:
                gc.enable()
        launches = COUNTERS["launches"] - before
        COUNTERS["launches"] = before          # captured, not run
        if self._graph_pool is None:
            self._graph_pool = graph.pool()
        if self._graph_event is None:
            self._graph_event = torch.cuda.Event()
            self._graph_event.record()
        return host, dev, graph, out, launches, shared

    def capture_decode_graphs(self, max_context: Optional[int] = None, batch_sizes: Optional[Sequence[int]] = None,
                              share_prefixes: bool = False) -> int:
        """Capture the decode graphs ahead of time, for every batch bucket (or the given ones) and
        every context bucket up to `max_context` (default: max_model_len), so that no step of a
        running service pays for a capture.  With `share_prefixes` also those of steps that read shared
        beginnings once, for every length of the keys behind them.  A graph is captured on a batch of padding rows, which
        write nothing, so live requests are not disturbed.  Returns the number of graphs captured."""
        if not self.graph_batch_sizes or self.device.type != "cuda" or not getattr(self.model, "graph_safe", True):
            return 0
        self._apply_launch_mode()
        limit = min(max_context or self.max_model_len, self.max_model_len)
        ctx_buckets, b = [], self._ctx_bucket(1)
        while True:
            ctx_buckets.append(b)
            if b >= limit:
                break
            b = self._ctx_bucket(b + 1)
        made = 0
        for bucket in (batch_sizes or self.graph_batch_sizes):
            if bucket not in self.graph_batch_sizes:
                raise SchedulerError(f"{bucket} is not one of the graph batch sizes {self.graph_batch_sizes}")
            for ctx_limit in ctx_buckets:
                if (bucket, ctx_limit, 0) not in self._graphs:
                    # a first, uncaptured run of the padded batch: it loads the kernel libraries
                    # and lets the GEMM library choose its algorithms outside the capture
                    ctx = self.pack([], [], pad_to=bucket, buffers=self._graph_buffers(bucket), ctx_limit=ctx_limit)
                    self.model.compute_logits(self.model.forward(ctx, self.cache), ctx)
                    self._graphs[(bucket, ctx_limit, 0)] = self._capture(bucket, ctx_limit)
                    made += 1
                for own_limit in ctx_buckets if share_prefixes else ():
                    if own_limit > ctx_limit or (bucket, ctx_limit, own_limit) in self._graphs or not self._may_share(bucket, ctx_limit):
                        continue
                    state = self._capture(bucket, ctx_limit, own_limit)
                    if not state[-1].used:
                        self._key_bytes = 0            # no layer reads beginnings once
                        break
                    self._graphs[(bucket, ctx_limit, own_limit)] = state
                    made += 1
        return made

    def finish(self, req_id: Hashable) -> None:
        """Give back everything the request holds."""
        if self.cache.has(req_id):
            self.cache.free(req_id)
