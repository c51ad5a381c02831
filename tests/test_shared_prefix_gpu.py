"""Attention of sequences that begin with the same cached tokens, and the tables of a step built on the device."""
from __future__ import annotations

import math
import random

import pytest
import torch

from rvllm_b200.errors import KernelError
from rvllm_b200.kernels import AttentionMeta, SharedPrefixes, StepPrefixes, get_library

pytestmark = pytest.mark.gpu

F64 = torch.float64


def lib():
    return get_library("cuda:0")


def make(groups, singles, nh, nkv, hd, page, dtype, seed=0, own=(1, 40), stale="nan", share="pages", max_blocks=None):
    """A step: `groups` = [(members, prefix tokens)], `singles` sequences alone; own lengths drawn from `own` (a list: as given).
    Slots that no sequence's tokens fill hold `stale`.  share "pages": a group's whole pages have several holders."""
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    order = [g for g, (n, _) in enumerate(groups) for _ in range(n)] + [-1] * singles
    rng.shuffle(order)
    B = len(order)
    prefix = [p for _, p in groups]
    own_lens = list(own) if isinstance(own, list) else [rng.randint(*own) for _ in order]
    ctx = [(prefix[g] if g >= 0 else 0) + n for g, n in zip(order, own_lens)]
    used = [(c + page - 1) // page for c in ctx]
    total = sum(used) + sum(p // page for p in prefix) + 5
    perm = torch.randperm(total, generator=gen).tolist()
    cache = torch.full((total, 2, nkv, page, hd), float(stale), dtype=torch.float32)
    MB = max_blocks or max(max(used), 1)
    table = torch.full((B, MB), -1, dtype=torch.int32)
    shared_kv = [torch.randn(2, nkv, p, hd, generator=gen) for p in prefix]
    shared_pages = {}
    kv = []
    for b, g in enumerate(order):
        mine = torch.randn(2, nkv, own_lens[b], hd, generator=gen)
        full = torch.cat([shared_kv[g], mine], 2) if g >= 0 else mine
        kv.append(full)
        for j in range(used[b]):
            key = (g, j)
            if share == "pages" and g >= 0 and (j + 1) * page <= prefix[g] and key in shared_pages:
                table[b, j] = shared_pages[key]
                continue
            pg = perm.pop()
            if g >= 0 and (j + 1) * page <= prefix[g]:
                shared_pages[key] = pg
            table[b, j] = pg
            hi = min(ctx[b], (j + 1) * page)
            if hi > j * page:
                cache[pg, :, :, :hi - j * page] = full[:, :, j * page:hi]
    q = torch.randn(B, nh * hd, generator=gen) * 2.0
    q, cache = q.to(dtype), cache.to(dtype)
    kv = [x.to(dtype).to(F64) for x in kv]
    meta = AttentionMeta(table.cuda(), torch.arange(B + 1, dtype=torch.int32).cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(),
                         torch.arange(B, dtype=torch.int32).cuda(), None, B, 1, max(ctx), page, B)
    plan = [([b for b, x in enumerate(order) if x == g], prefix[g]) for g in range(len(groups))]
    return dict(q=q.cuda(), cache=cache.cuda(), meta=meta, plan=plan, kv=kv, ctx=ctx, dims=(nh, nkv, hd), dtype=dtype)


def plain(s, scale, softcap=None, sinks=None, gate=None):
    """(attention, bound on the error) in 64 bits.

    The bound: a score is a sum of hd products in 32 bits (off by at most hd 2^-24 of the sum of their absolute values, and by the
    tanh's and exponential's few 2^-22 of the score), which moves every weight by that much, up and down, in numerator and
    denominator; bfloat16 weights are off by half a step of their type (2^-8), the result by another."""
    nh, nkv, hd = s["dims"]
    per = nh // nkv
    out, tol = [], []
    for b, kv in enumerate(s["kv"]):
        q = s["q"][b].cpu().to(F64).view(nkv, per, hd)
        n = s["ctx"][b]
        k, v = kv[0][:, :n], kv[1][:, :n]
        raw = torch.einsum("gph,gkh->gpk", q, k) * scale
        x = softcap * torch.tanh(raw / softcap) if softcap else raw
        size = torch.einsum("gph,gkh->gpk", q.abs(), k.abs()) * scale
        off = (hd + 4) * 2.0 ** -24 * (size.amax(-1) if n else torch.zeros(nkv, per, dtype=F64)) + 2.0 ** -20 * (softcap or 0) + 2.0 ** -20
        if sinks is not None:
            x = torch.cat([x, sinks.cpu().to(F64).view(nkv, per, 1)], -1)
        if x.shape[-1] == 0:
            out.append(torch.zeros(nh, hd, dtype=F64)); tol.append(torch.zeros(nh, hd, dtype=F64))
            continue
        w = torch.softmax(x, -1)[..., :n]
        o, a = w @ v, w @ v.abs()
        step = 2.0 ** -8 if s["dtype"] == torch.bfloat16 else 2.0 ** -24
        t = (2 * off[..., None] + (n + 16) * 2.0 ** -24 + step) * a + step * o.abs()
        f = gate[b].cpu().to(F64).view(nkv, per, 1) if gate is not None else 1.0
        out.append((o * f).reshape(nh, hd)); tol.append((t * f).reshape(nh, hd) + 1e-30)
    return torch.stack(out).flatten(1), torch.stack(tol).flatten(1)


def run(s, softcap=None, sinks=None, gate=None, max_own=None, scale=None, meta=None, shared=None):
    nh, nkv, hd = s["dims"]
    shared = shared or SharedPrefixes(s["plan"], len(s["ctx"]), nh, nkv, "cuda")
    return lib().shared_prefix_attention(s["q"], s["cache"], meta or s["meta"], shared, nh, nkv, hd, scale or hd ** -0.5, softcap, sinks, gate,
                                         max_own=max_own)


def check(s, **kw):
    got = run(s, **kw).cpu().to(F64)
    lib().raise_on_abort()
    want, tol = plain(s, kw.get("scale") or s["dims"][2] ** -0.5, kw.get("softcap"), kw.get("sinks"), kw.get("gate"))
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / tol.clamp(min=1e-30))
    assert float(over.max()) <= 1.0, f"{float(over.max()):.2f} times the bound at {divmod(int(over.argmax()), want.shape[1])}"


CASES = [
    # groups, singles, heads, kv heads, head size, page, own lengths
    ([(2, 33)], 0, 14, 2, 64, 16, (1, 9)),
    ([(2, 1)], 0, 4, 4, 64, 16, (1, 1)),                          # a prefix of one token
    ([(8, 128)], 0, 28, 4, 128, 16, (1, 70)),                     # tiles that end with the prefix
    ([(5, 129)], 1, 32, 8, 128, 8, (1, 200)),
    ([(40, 200)], 0, 32, 8, 128, 16, (1, 30)),                    # two row tiles, the second partly filled
    ([(19, 64), (3, 100), (2, 700)], 4, 28, 4, 128, 32, (1, 130)),   # 126 rows to a tile
    ([(3, 65)], 2, 8, 1, 64, 64, (1, 300)),
    ([(2, 300)], 0, 128, 1, 128, 16, (1, 20)),                    # 128 heads on one
    ([(3, 90)], 1, 16, 16, 128, 128, (1, 20)),                    # pages larger than a tile
    ([(64, 1000)], 3, 16, 4, 128, 16, (1, 64)),
    ([(300, 77)], 0, 4, 2, 64, 16, (1, 5)),                       # hundreds of sequences, few keys each
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_64_bits(case, dtype):
    groups, singles, nh, nkv, hd, page, own = CASES[case]
    if dtype == torch.float32 and case in (9, 10):
        groups = [(n // 4, p) for n, p in groups]
    check(make(groups, singles, nh, nkv, hd, page, dtype, seed=case, own=own))


@pytest.mark.parametrize("dtype,hd,page", [(torch.bfloat16, 32, 16), (torch.bfloat16, 80, 16), (torch.bfloat16, 256, 16), (torch.bfloat16, 128, 24),
                                           (torch.bfloat16, 64, 4), (torch.float32, 20, 16), (torch.float32, 132, 7), (torch.float32, 256, 1)])
def test_sizes_of_the_plain_kernels(dtype, hd, page):
    check(make([(6, 75), (2, 10)], 1, 6, 2, hd, page, dtype, seed=hd, own=(1, 50)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("own", [[0, 0, 0], [0, 1, 70], [1, 64, 65]])
def test_nothing_behind_the_prefix(dtype, own):
    """A context that ends with the prefix: the keys behind it are none."""
    check(make([(3, 96)], 0, 8, 2, 64, 16, dtype, own=own))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_rows_that_stand_for_no_request(dtype):
    """A context length of 0 gives zeros, inside a group or outside; a context inside the prefix sees no further."""
    s = make([(4, 100)], 2, 8, 2, 64, 16, dtype, seed=3, own=(1, 30))
    members = s["plan"][0][0]
    outside = [b for b in range(6) if b not in members][0]
    ctx = list(s["ctx"])
    ctx[members[1]], ctx[members[2]], ctx[outside] = 0, 37, 0
    s["ctx"] = ctx
    s["meta"].ctx_lens.copy_(torch.tensor(ctx, dtype=torch.int32))
    out = run(s)
    assert float(out[members[1]].abs().max()) == 0.0 and float(out[outside].abs().max()) == 0.0
    check(s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("stale", ["nan", "inf", "-3.4e38"])
@pytest.mark.parametrize("seqs", [4, 70])
def test_what_earlier_requests_left(dtype, stale, seqs):
    """Slots behind a prefix's and a sequence's last token hold anything: nothing of it is seen (seqs 70: the evenly cut kernel)."""
    check(make([(seqs, 70)], 2, 8, 4, 64, 16, dtype, seed=5, own=(1, 90), stale=stale, share="copies"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("seqs", [5, 80])
@pytest.mark.parametrize("which", ["cap", "sink", "gate", "all"])
def test_cap_sink_gate(dtype, which, seqs):
    s = make([(seqs, 150)], 1, 16, 4, 128, 16, dtype, seed=9, own=(0, 60))
    gen = torch.Generator().manual_seed(1)
    sinks = (torch.randn(16, generator=gen) * 3).cuda() if which in ("sink", "all") else None
    gate = torch.rand(seqs + 1, 16, generator=gen).cuda() if which in ("gate", "all") else None
    check(s, softcap=5.0 if which in ("cap", "all") else None, sinks=sinks, gate=gate)


def test_scores_far_apart():
    """Scores that climb along the prefix make the running maximum move in every tile; later ones fall far below it."""
    for dtype in (torch.bfloat16, torch.float32):
        s = make([(33, 900)], 1, 8, 2, 128, 16, dtype, seed=2, own=(1, 100))
        s["q"].mul_(6)
        check(s)


def test_max_own_sizes_the_launch_only():
    s = make([(6, 500)], 0, 32, 8, 128, 16, torch.bfloat16, seed=4, own=(1, 300))
    outs = [run(s, max_own=n).float() for n in (None, 1, 64, 300, 5000)]
    for o in outs[1:]:
        assert float((o - outs[0]).abs().max()) <= 2.0 ** -7 * float(outs[0].abs().max())
    check(s, max_own=1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_what_is_not_a_number_stays_so(dtype):
    """A query of NaN, and keys of NaN or infinity that a sequence sees, give NaN to that sequence (or its heads) and to no other."""
    s = make([(5, 70)], 2, 8, 2, 64, 16, dtype, seed=3, own=[9, 20, 33, 4, 18, 40, 7])
    nh, nkv, hd = s["dims"]
    s["q"][1] = float("nan")
    for b, value in ((3, float("nan")), (4, float("inf"))):
        at = s["ctx"][b] - 1                         # its own last key, of one kv head
        s["cache"][s["meta"].block_tables[b, at // 16], 0, 1, at % 16] = value
    got = run(s).view(7, nkv, nh // nkv, hd).cpu()
    lib().raise_on_abort()
    want = torch.zeros(7, nkv, dtype=torch.bool)
    want[1] = True
    want[3, 1] = want[4, 1] = True
    assert torch.equal(got.isnan().all(-1).all(-1), want) and torch.equal(got.isnan().any(-1).any(-1), want)


def test_long_prefix_in_many_ranges():
    s = make([(3, 9001)], 1, 8, 2, 128, 16, torch.bfloat16, seed=6, own=(1, 40))
    check(s)
    check(make([(3, 9001)], 1, 8, 2, 64, 16, torch.bfloat16, seed=6, own=(1, 40)))


def test_more_sequences_than_the_list_of_pieces_has_room_for():
    check(make([(2100, 33)], 2, 2, 1, 64, 16, torch.bfloat16, seed=8, own=(1, 20)))
    check(make([(2040, 33)], 2, 2, 1, 64, 16, torch.bfloat16, seed=8, own=(1, 20)))


def test_without_groups_it_is_the_paged_attention():
    s = make([], 5, 32, 8, 128, 16, torch.bfloat16, own=(1, 300), stale="0")
    nh, nkv, hd = s["dims"]
    want = lib().paged_attention(s["q"], s["cache"], s["meta"], nh, nkv, hd, hd ** -0.5, None)
    assert torch.equal(run(s), want)
    alone = SharedPrefixes([([2], 100), ([0, 1], 0)], 5, nh, nkv, "cuda")
    assert alone.capacity == (0, 0) and torch.equal(run(s, shared=alone), want)


@pytest.mark.parametrize("dtype,hd,page,once", [(torch.bfloat16, 96, 16, False), (torch.bfloat16, 80, 16, False), (torch.bfloat16, 256, 16, False),
                                                (torch.bfloat16, 128, 4, False), (torch.bfloat16, 128, 16, True), (torch.float32, 96, 16, True)])
def test_which_steps_paged_attention_reads_once(dtype, hd, page, once, monkeypatch):
    """Heads and pages that the tensor-core kernel of shared beginnings does not take stay with the one that takes each sequence for itself."""
    s = make([(6, 96)], 1, 8, 2, hd, page, dtype, seed=hd, own=(1, 50), stale="0")
    calls, original = [], lib().shared_prefix_attention
    monkeypatch.setattr(lib(), "shared_prefix_attention", lambda *a, **kw: (calls.append(1), original(*a, **kw))[1])
    call = lambda: lib().paged_attention(s["q"], s["cache"], s["meta"], 8, 2, hd, hd ** -0.5, None)  # noqa: E731
    want = call()
    s["meta"].shared = StepPrefixes(s["plan"], 7, "cuda")
    got = call()
    assert len(calls) == once and (once or torch.equal(got, want))
    exact, tol = plain(s, hd ** -0.5)
    assert float(((got.cpu().to(F64) - exact).abs() / tol).max()) <= 1.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_scales_that_only_paged_attention_takes(dtype, scale):
    """A scale that is not positive (some configurations allow any number) is no reason for a step with shared beginnings to fail."""
    s = make([(6, 96)], 1, 8, 2, 64, 16, dtype, seed=2, own=(1, 50), stale="0")
    call = lambda: lib().paged_attention(s["q"], s["cache"], s["meta"], 8, 2, 64, scale, None)  # noqa: E731
    want = call()
    s["meta"].shared = StepPrefixes(s["plan"], 7, "cuda")
    assert torch.equal(call(), want)


def test_pages_that_do_not_exist_are_not_read():
    """Entries beyond the cache or negative inside the prefix: no result is promised, and nothing outside the cache is touched."""
    for dtype in (torch.bfloat16, torch.float32):
        s = make([(3, 200)], 0, 8, 2, 64, 16, dtype, own=(1, 20), stale="0")
        t = s["meta"].block_tables
        t[:, 3] = -1
        t[:, 5] = s["cache"].shape[0] + 7
        assert run(s).shape == s["q"].shape
        torch.cuda.synchronize()
        lib().raise_on_abort()


def test_captured_and_replayed_with_other_groups():
    """A graph holds the launches; lengths, tables and groups are what its buffers hold when it is replayed."""
    nh, nkv, hd, B = 16, 4, 128, 12
    a = make([(12, 130)], 0, nh, nkv, hd, 16, torch.bfloat16, seed=1, own=(1, 30), max_blocks=64)
    b = make([(4, 500), (5, 77)], 3, nh, nkv, hd, 16, torch.bfloat16, seed=2, own=(1, 30), max_blocks=64)
    cap = (6, 80)
    plans = [SharedPrefixes(s["plan"], B, nh, nkv, "cuda", capacity=cap) for s in (a, b)]
    shared = SharedPrefixes([], B, nh, nkv, "cuda", capacity=cap)
    pages = max(a["cache"].shape[0], b["cache"].shape[0])
    cache = torch.zeros((pages, *a["cache"].shape[1:]), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros_like(a["q"])
    table, ctx = torch.full((B, 64), -1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    meta = AttentionMeta(table, a["meta"].cu_seqlens, ctx, a["meta"].token_seq, None, B, 1, 1024, 16, B)

    def fill(s, plan):
        cache[:s["cache"].shape[0]] = s["cache"]; q.copy_(s["q"]); table.copy_(s["meta"].block_tables); ctx.copy_(s["meta"].ctx_lens)
        shared.device_ints.copy_(plan.device_ints)

    call = lambda: lib().shared_prefix_attention(q, cache, meta, shared, nh, nkv, hd, hd ** -0.5, max_own=64)  # noqa: E731
    fill(a, plans[0])
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for s, plan in ((a, plans[0]), (b, plans[1]), (a, plans[0])):
        fill(s, plan)
        graph.replay()
        want, tol = plain(s, hd ** -0.5)
        assert float(((out.cpu().to(F64) - want).abs() / tol).max()) <= 1.0
    shared.device_ints.zero_()                     # no group: every sequence is all its own ... which the array has to say
    shared.device_ints[4 + B:4 + 2 * B] = -1
    graph.replay()
    want, tol = plain(a, hd ** -0.5)
    assert float(((out.cpu().to(F64) - want).abs() / tol).max()) <= 1.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_refilled_with_wider_groups(dtype):
    """A layout with a capacity, made for two sequences behind a short prefix, serves sixteen: every row of their tile is computed."""
    s = make([(16, 64)], 0, 16, 4, 128, 16, dtype, seed=21, own=(1, 30))
    shared = SharedPrefixes([([0, 1], 64)], 16, 16, 4, "cuda", capacity=(3, 12))
    check(s, shared=shared)
    shared.refill(s["plan"])
    check(s, shared=shared)
    shared.refill([])
    check(s, shared=shared)


def test_groups_are_sent_while_the_device_is_busy():
    """New groups and new layouts travel on the stream: the host does not wait for what was launched before them, and one after the
    other arrive as they were."""
    plans = [[(list(range(n)), 64 * n), (list(range(n, 60)), 100)] for n in (3, 20, 41)]
    make_one = lambda plan: SharedPrefixes(plan, 64, 32, 8, "cuda", capacity=(20, 80))  # noqa: E731
    want = [make_one(p).device_ints.cpu() for p in plans]
    shared, step = make_one([]), StepPrefixes([], 64, "cuda", 4)
    layout = step.layout(32, 8)
    torch.cuda.synchronize()
    copies = []
    torch.cuda._sleep(200_000_000)                   # about a tenth of a second
    busy = torch.cuda.Event()
    busy.record()
    for p in plans:
        shared.refill(p)
        copies.append(shared.device_ints.clone())
    step.set_groups(plans[0])
    late = make_one(plans[2])
    assert not busy.query(), "the host waited for the device"
    torch.cuda.synchronize()
    assert all(torch.equal(c.cpu(), w) for c, w in zip(copies, want)) and torch.equal(late.device_ints.cpu(), want[2])
    assert layout.own_start.tolist() == want[0][4:68].tolist()


def test_groups_are_not_changed_inside_a_capture():
    s = make([(12, 130)], 0, 16, 4, 128, 16, torch.bfloat16, seed=1, own=(1, 30))
    shared, step = SharedPrefixes(s["plan"], 12, 16, 4, "cuda", capacity=(6, 80)), StepPrefixes(s["plan"], 12, "cuda", 4)
    want = run(s, shared=shared).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: shared.refill([]), lambda: SharedPrefixes(s["plan"], 12, 16, 4, "cuda"), lambda: step.layout(16, 4)):
            with pytest.raises(KernelError, match="capture"):
                call()
        out = run(s, shared=shared)
    graph.replay()
    assert torch.equal(out, want)
    shared.refill([([0, 1], 64)])                    # the refused calls left nothing behind
    assert shared.own_start.tolist() == [64, 64] + [0] * 10 and step.layout(16, 4).own_start.tolist() == [130] * 12


def test_on_another_stream_and_twice_at_once():
    a = make([(30, 600)], 2, 32, 8, 128, 16, torch.bfloat16, seed=11, own=(1, 100))
    b = make([(30, 333)], 2, 32, 8, 128, 16, torch.bfloat16, seed=12, own=(1, 100))
    shared = [SharedPrefixes(s["plan"], 32, 32, 8, "cuda") for s in (a, b)]
    want = [run(s, shared=p).clone() for s, p in zip((a, b), shared)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for i, (s, p) in enumerate(zip((a, b), shared)):
            with torch.cuda.stream(streams[i]):
                got[i] = run(s, shared=p)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_a_layout_that_is_still_on_its_way_to_another_stream(dtype):
    """Made, and changed, on a busy stream and used at once on another: the call waits for the copy on the device."""
    s = make([(12, 130)], 1, 16, 4, 128, 16, dtype, seed=1, own=(1, 30))
    exact = SharedPrefixes(s["plan"], 13, 16, 4, "cuda")
    roomy = SharedPrefixes([], 13, 16, 4, "cuda", capacity=(6, 80))
    roomy.refill(s["plan"])
    want = [run(s, shared=exact).clone(), run(s, shared=roomy).clone()]
    roomy.refill([])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda._sleep(100_000_000)                   # about a twentieth of a second
    late = SharedPrefixes(s["plan"], 13, 16, 4, "cuda")
    roomy.refill(s["plan"])
    with torch.cuda.stream(side):
        got = [run(s, shared=late), run(s, shared=roomy)]
    torch.cuda.synchronize()
    lib().raise_on_abort()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_refusals():
    s = make([(4, 50)], 1, 8, 2, 64, 16, torch.bfloat16, own=(1, 20))
    nh, nkv, hd = s["dims"]
    shared = SharedPrefixes(s["plan"], 5, nh, nkv, "cuda")
    call = lambda q=s["q"], c=s["cache"], m=s["meta"], p=shared, h=(nh, nkv, hd), scale=0.125, **kw: lib().shared_prefix_attention(q, c, m, p, *h, scale, **kw)  # noqa: E731
    call()
    m = s["meta"]
    two = AttentionMeta(m.block_tables, m.cu_seqlens, m.ctx_lens, m.token_seq, None, 5, 2, 100, 16, 4)
    bad = [dict(q=s["q"][:4]), dict(q=s["q"].half()), dict(q=s["q"].float()), dict(q=s["q"].view(5, 2, 256)[:, 0]), dict(q=s["q"].cpu()),
           dict(c=s["cache"][:, :1].contiguous()), dict(c=s["cache"].transpose(2, 3)), dict(m=two), dict(h=(8, 4, 64)), dict(h=(8, 2, 32)),
           dict(p=SharedPrefixes(s["plan"], 6, nh, nkv, "cuda")), dict(p=SharedPrefixes(s["plan"], 5, 2, 2, "cuda")),
           dict(p=SharedPrefixes(s["plan"], 5, nh, nkv, "cpu")), dict(sinks=torch.zeros(3, device="cuda")), dict(sinks=torch.zeros(8)),
           dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")), dict(gate=torch.zeros(5, 7, device="cuda")), dict(gate=torch.zeros(5, 8, device="cuda", dtype=torch.bfloat16))]
    for kw in bad:
        with pytest.raises(KernelError):
            call(**kw)


# ------------------------------------------------------------------------------------------------------------ tables
def plain_tables(table, rows, held, starts, q_lens, new, spans, T, MB, page):
    G, R, W = table.shape
    B = len(rows)
    table = table.clone()
    bt = torch.full((G, B, MB), -1, dtype=torch.int32)
    slot = torch.full((G, T), -1, dtype=torch.int32)
    pos, seq = torch.zeros(T, dtype=torch.int32), torch.full((T,), -1, dtype=torch.int32)
    cu, ctx = [0], []
    at = 0
    for g in range(G):
        t = 0
        for b in range(B):
            used = min(W, -(-(starts[b] + q_lens[b]) // page)) if rows[b] >= 0 else 0
            for j in range(held[g][b], used):
                table[g, rows[b], j] = new[at]
                at += 1
            window, chunk = spans[g]
            first = max(0, starts[b] - window + 1) if window else 0
            first = max(first, starts[b] // chunk * chunk if chunk else 0)
            for j in range(first // page, min(used, MB)):
                bt[g, b, j] = table[g, rows[b], j]
            for i in range(q_lens[b]):
                p = starts[b] + i if rows[b] >= 0 else 0
                if rows[b] >= 0:
                    slot[g, t] = table[g, rows[b], p // page] * page + p % page
                pos[t], seq[t] = p, b
                t += 1
            if g == 0:
                cu.append(cu[-1] + q_lens[b])
                ctx.append(starts[b] + q_lens[b] if rows[b] >= 0 else 0)
    return table, (bt, slot, pos, seq, torch.tensor(cu, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32))


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


TABLES = [  # sequences, groups, page, longest context, share of prompts, padding rows, spans, tokens to spare
    (1, 1, 16, 1, 0.0, 0, [(0, 0)], 0),
    (1, 1, 16, 40, 1.0, 0, [(0, 0)], 0),
    (8, 1, 16, 2000, 0.0, 3, [(0, 0)], 0),
    (7, 2, 1, 90, 0.5, 0, [(0, 0), (17, 0)], 5),
    (33, 3, 32, 3000, 0.3, 1, [(0, 0), (100, 0), (0, 256)], 0),
    (300, 2, 8, 500, 0.1, 44, [(0, 64), (31, 0)], 3),
    (1025, 1, 16, 700, 0.02, 0, [(0, 0)], 0),
]


@pytest.mark.parametrize("case", range(len(TABLES)))
@pytest.mark.parametrize("own_out", [False, True])
def test_step_tables(case, own_out):
    from rvllm_b200.kernels import StepTables
    B, G, page, longest, prompts, pads, spans, spare = TABLES[case]
    rng = random.Random(case)
    R = B + 3
    rows = rng.sample(range(R), B)
    for i in range(B - pads, B):
        rows[i] = -1
    q = [rng.choice((0, 2, 3, 70)) if rng.random() < prompts else 1 for _ in range(B)]
    starts = [rng.randint(0, longest - 1) for _ in range(B)]
    used = [-(-(s + n) // page) if r >= 0 else 0 for s, n, r in zip(starts, q, rows)]
    # what a row holds already: the blocks of its earlier tokens, or - a request that just took over another's leading pages - none
    held = [[min(u, -(-s // page)) if rng.random() < 0.8 else 0 for u, s in zip(used, starts)] for _ in range(G)]
    W, T = max(used) + 2, sum(q) + spare
    MB = max(max(used), 1) + (case % 2)
    n_new = sum(u - h for row in held for u, h in zip(used, row))
    new = [rng.randrange(1, 1 << 20) for _ in range(n_new)]
    table = torch.randint(0, 1 << 20, (G, R, W), dtype=torch.int32)
    want_table, want = plain_tables(table, rows, held, starts, q, new, spans, T, MB, page)
    dev = table.cuda()
    out = StepTables(*(torch.full(w.shape, 77, dtype=torch.int32, device="cuda") for w in want)) if own_out else None
    args = (i32(rows), i32(held), i32(starts), i32(q), i32(new), i32(spans), T, MB, page)
    got = lib().step_tables(dev, *args, out=out)
    assert own_out is (got is out)
    for _ in range(2):                              # a second call on what the first left gives the same
        for w, x in zip(want, (got.block_tables, got.slot_mapping, got.positions, got.token_seq, got.cu_seqlens, got.ctx_lens)):
            assert torch.equal(x.cpu(), w)
        assert torch.equal(dev.cpu(), want_table)
        got = lib().step_tables(dev, *args, out=out)


def test_step_tables_check_what_the_device_holds():
    """Rows, lengths and counts out of range are cut off or count as absent: nothing outside the tensors is read or written."""
    table = torch.zeros((1, 4, 3), dtype=torch.int32, device="cuda")
    guard = torch.full((1, 2, 5), 9, dtype=torch.int32, device="cuda")
    got = lib().step_tables(table, i32([2, 9]), i32([[-4, 0]]), i32([40, -3]), i32([30, 5]), i32([5]), i32([[0, 0]]), 20, 5, 16)
    torch.cuda.synchronize()
    # the row of three blocks takes the one page there is; the two that are missing, and the sequence without a row, are absent
    assert table[0, 2].tolist() == [5, -1, -1] and table[0, [0, 1, 3]].abs().sum() == 0
    assert got.block_tables.tolist() == [[[5, -1, -1, -1, -1], [-1] * 5]] and got.ctx_lens.tolist() == [70, 0]
    assert got.slot_mapping.tolist() == [[-1] * 20] and guard.eq(9).all()


def test_step_tables_with_lengths_past_31_bits():
    """Sums that leave 32-bit integers: every tensor lies between guards, and these stay as they are."""
    from rvllm_b200.kernels import StepTables
    top = 2 ** 31 - 1
    many = 600                                       # (more than a CTA takes by itself)
    for starts, q, held in (([top] * 5, [top] * 5, [top] * 5), ([top - 3, 0, top, 7, 1], [9, top, top, 3, 1], [0, top, -top, 3, 1]),
                            ([1] * many, [top // 2] * many, [top] * many)):
        B, T, MB, W = len(starts), 40, 6, 4
        shapes = [(1, B, W), (1, B, MB), (1, T), (T,), (T,), (B + 1,), (B,)]
        room = torch.full((sum(math.prod(s) + 64 for s in shapes) + 64,), 123456789, dtype=torch.int32, device="cuda")
        views, at = [], 64
        for s in shapes:
            views.append(room[at:at + math.prod(s)].view(s))
            at += math.prod(s) + 64
        lib().step_tables(views[0], i32(list(range(B))), i32([held]), i32(starts), i32(q), i32([3, 4]), i32([[0, 0]]), T, MB, 16, out=StepTables(*views[1:]))
        at = 0
        for s in shapes:
            assert room[at:at + 64].eq(123456789).all()
            at += math.prod(s) + 64
        assert room[at:].eq(123456789).all()


@pytest.mark.parametrize("rows,held,starts,q", [
    ([2, 9], [-4, 0], [40, -3], [30, 5]), ([-7, 2 ** 31 - 1], [0, 0], [5, 5], [3, 3]), ([0, 3], [99, -99], [0, 47], [1, 1]),
    ([1, 2], [0, 0], [4000, 46], [5, 9]), ([3, 0], [3, 3], [-50, 100], [90, -90]), ([-2 ** 31, 3], [-2 ** 31, 2 ** 31 - 1], [-2 ** 31, 0], [-2 ** 31, 48])])
def test_step_tables_write_inside_their_tensors(rows, held, starts, q):
    """Rows, held entries, starts and lengths out of range: the page table and every output lie between guards, and these stay as they are;
    so do the rows of the page table that no sequence of the step owns."""
    from rvllm_b200.kernels import StepTables
    R, W, MB, T = 4, 3, 5, 20
    shapes = [(1, R, W), (1, 2, MB), (1, T), (T,), (T,), (3,), (2,)]
    room = torch.full((sum(math.prod(s) + 64 for s in shapes) + 64,), 123456789, dtype=torch.int32, device="cuda")
    views, at = [], 64
    for s in shapes:
        views.append(room[at:at + math.prod(s)].view(s))
        at += math.prod(s) + 64
    views[0].zero_()
    lib().step_tables(views[0], i32(rows), i32([held]), i32(starts), i32(q), i32([5, 6]), i32([[0, 0]]), T, MB, 16, out=StepTables(*views[1:]))
    at = 0
    for s in shapes:
        assert room[at:at + 64].eq(123456789).all()
        at += math.prod(s) + 64
    assert room[at:].eq(123456789).all()
    others = [r for r in range(R) if r not in rows]
    assert views[0][0, others].eq(0).all() and views[0].ge(-1).all() and views[0].le(6).all()
    assert views[1].ge(-1).all() and views[1].le(6).all()


def test_step_tables_captured():
    table = torch.zeros((1, 2, 8), dtype=torch.int32, device="cuda")
    rows, held, starts, q, new, spans = i32([1, 0]), i32([[0, 0]]), i32([0, 0]), i32([1, 1]), i32([3, 4]), i32([[0, 0]])
    call = lambda: lib().step_tables(table, rows, held, starts, q, new, spans, 2, 4, 4)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    starts.copy_(i32([4, 3])); held.copy_(i32([[1, 1]])); new.copy_(i32([6, 0]))
    graph.replay()
    assert out.block_tables.tolist() == [[[3, 6, -1, -1], [4, -1, -1, -1]]] and out.slot_mapping.tolist() == [[24, 19]]
    assert out.ctx_lens.tolist() == [5, 4] and table[0].tolist()[1][:2] == [3, 6]


def test_tables_are_settled_while_any_library_launches_early(monkeypatch):
    """The switch of a single source file says how its own kernels are launched, not whether those behind the tables are launched early."""
    import struct
    k = lib()
    k.set_pdl(True)
    one = (torch.zeros((1, 2, 4), dtype=torch.int32, device="cuda"), i32([0]), i32([[0]]), i32([0]), i32([1]), i32([1]), i32([[0, 0]]), 1, 4, 16)
    k.step_tables(*one)
    seen, original = [], k._entries["tables"]
    monkeypatch.setitem(k._entries, "tables", lambda block: (seen.append(struct.unpack_from("=i", block, 13 * 8 + 8 * 4 + 8)[0]), original(block))[1])
    monkeypatch.setattr(k, "pdl", True)
    for alone in ((), ("step_tables.cu",)):
        monkeypatch.setattr(k, "no_pdl_for", alone)
        k._lib("step_tables.cu").rv_set_pdl(0 if alone else 1)
        k.step_tables(*one)
        k.step_tables(*one, settle=False)
    monkeypatch.setattr(k, "pdl", False)
    k.step_tables(*one)
    k._lib("step_tables.cu").rv_set_pdl(1)
    torch.cuda.synchronize()
    assert seen == [1, 0, 1, 0, 0]


def test_attention_right_behind_the_tables():
    """Tables that change from call to call, read by the launch right behind, which starts early where the library launches it so."""
    s = make([], 40, 32, 8, 128, 16, torch.bfloat16, seed=3, own=(300, 900), stale="0")
    B, real, ctx = 40, s["meta"].block_tables, s["meta"].ctx_lens
    MB, W = real.shape[1], real.shape[1] + 1
    q_lens, held, spans = i32([1] * B), i32([[0] * B]), i32([[0, 0]])
    orders = [torch.randperm(B, generator=torch.Generator().manual_seed(i)) for i in range(6)]
    table = torch.full((1, B, W), -1, dtype=torch.int32, device="cuda")
    want = lib().paged_attention(s["q"], s["cache"], s["meta"], 32, 8, 128, 128 ** -0.5, None)
    steps = []
    for order in orders:                             # sequence i of a step is sequence order[i] of the cache
        lens = [s["ctx"][int(b)] for b in order]
        new = torch.cat([real[int(b), :(n + 15) // 16] for b, n in zip(order, lens)])
        steps.append((order.cuda(), s["q"][order.cuda()].contiguous(), i32([n - 1 for n in lens]), new.contiguous()))
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for order, q, starts, new in steps:
            t = lib().step_tables(table, i32(list(range(B))), held, starts, q_lens, new, spans, B, MB, 16)
            meta = AttentionMeta(t.block_tables[0], t.cu_seqlens, t.ctx_lens, t.token_seq, t.slot_mapping[0], B, 1, int(max(s["ctx"])), 16, B)
            got.append((order, lib().paged_attention(q, s["cache"], meta, 32, 8, 128, 128 ** -0.5, None)))
    torch.cuda.synchronize()
    for order, out in got:
        assert torch.equal(out, want[order])


def test_step_tables_refusals():
    good = dict(page_table=torch.zeros((1, 2, 4), dtype=torch.int32, device="cuda"), rows=i32([0, 1]), held=i32([[0, 0]]), starts=i32([0, 0]),
                q_lens=i32([1, 1]), new_pages=i32([1, 2]), spans=i32([[0, 0]]), num_tokens=2, max_blocks=4, page_size=16)
    lib().step_tables(**good)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    for bad in (dict(rows=i32([0])), dict(held=i32([0, 0])), dict(held=i32([[0]])), dict(spans=i32([[0, 0], [0, 0]])), dict(max_blocks=0),
                dict(page_size=0), dict(num_tokens=-1), dict(starts=i32([0, 0]).long()), dict(q_lens=i32([1, 1]).cpu()),
                dict(page_table=torch.zeros((1, 4, 2), dtype=torch.int32, device="cuda").transpose(1, 2)),
                dict(rows=none, held=none.view(1, 0), starts=none, q_lens=none),
                dict(out=lib().step_tables(**{**good, "max_blocks": 5}))):
        with pytest.raises(KernelError):
            lib().step_tables(**{**good, **bad})
