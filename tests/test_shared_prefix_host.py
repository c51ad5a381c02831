"""The layout of shared prefixes, checked without a GPU."""
import random

import pytest
import torch

from rvllm_b200.errors import KernelError
from rvllm_b200.kernels import SharedPrefixes, StepPrefixes


def unpack(s):
    """The array as the kernels read it (csrc/shared_prefix.cuh)."""
    v, B = s.device_ints.tolist(), s.num_seqs
    tiles, items = s.capacity
    at = (4 + 3 * B + 2 * tiles + 3) // 4 * 4
    ranges = [v[at + 8 * i:at + 8 * i + 8] for i in range(items)]
    rows = {r[5]: r[2:5] for r in ranges[:v[0]]}
    return dict(items_used=v[0], tiles_used=v[1], own_start=v[4:4 + B], place=v[4 + B:4 + 2 * B], members=v[4 + 2 * B:4 + 3 * B],
                parts=[v[4 + 3 * B + 2 * i:4 + 3 * B + 2 * i + 2] for i in range(tiles)], tiles=rows, items=ranges, size=len(v))


@pytest.mark.parametrize("seed", range(12))
def test_every_row_and_key_once(seed):
    rng = random.Random(seed)
    nkv = rng.choice((1, 2, 4, 8))
    nh = nkv * rng.choice((1, 2, 4, 7, 32, 128))
    B = rng.randint(1, 300)
    free = list(range(B))
    rng.shuffle(free)
    groups = []
    while free and rng.random() < 0.8:
        n = rng.randint(1, min(len(free), 200))
        groups.append(([free.pop() for _ in range(n)], rng.choice((0, 1, 63, 64, 65, rng.randint(1, 40000)))))
    s = SharedPrefixes(groups, B, nh, nkv, "cpu")
    u = unpack(s)
    assert u["size"] == SharedPrefixes.ints(B, s.capacity)
    per = nh // nkv
    of = {m: (g, t) for g, (ms, t) in enumerate(groups) for m in ms if len(ms) > 1 and t > 0}
    rows = set()
    for b in range(B):
        if b not in of:
            assert u["own_start"][b] == 0 and u["place"][b] == -1
            continue
        tile, row = divmod(u["place"][b], 128)
        seq, first, count = u["tiles"][tile]
        assert of[b][1] == u["own_start"][b] and seq in groups[of[b][0]][0]
        assert row % per == 0 and row + per <= 128 and u["members"][first + row // per] == b and row // per < count
        rows.add((tile, row))
    assert len(rows) == len(of)
    for t in range(u["tiles_used"]):
        first, n = u["parts"][t]
        at = 0
        for lo, hi, seq, _, _, tile, _, _ in u["items"][first:first + n]:
            assert tile == t and lo == at and lo % 64 == 0 and lo < hi
            at = hi
        assert at == u["own_start"][u["tiles"][t][0]]
    assert u["items_used"] == sum(n for _, n in u["parts"][:u["tiles_used"]])


def test_ranges_fill_the_places_once():
    s = SharedPrefixes([(list(range(64)), 4096)], 64, 32, 8, "cpu")
    assert s.num_tiles == 2 and 0.6 * 148 < s.num_items * 8 <= 148
    s = SharedPrefixes([(list(range(4)), 32768)], 4, 32, 8, "cpu")
    assert 0.9 * 296 < s.num_items * 8 <= 296


def test_a_capacity_fixes_the_size():
    sizes = {SharedPrefixes(g, 8, 16, 4, "cpu", capacity=(3, 90)).device_ints.numel() for g in ([], [([0, 1], 50)], [([0, 1], 50), ([5, 3, 2], 700)])}
    assert len(sizes) == 1
    with pytest.raises(KernelError):
        SharedPrefixes([([0, 1], 5), ([2, 3], 5)], 8, 16, 4, "cpu", capacity=(1, 90))
    with pytest.raises(KernelError):
        SharedPrefixes([([0, 1], 5000)], 8, 16, 4, "cpu", capacity=(1, 2))


@pytest.mark.parametrize("groups", [[([0, 0], 5)], [([0, 1], 5), ([1, 2], 5)], [([0, 9], 5)], [([-1, 0], 5)], [([0, 1], -1)], [([0, 1], 2 ** 31)]])
def test_refused_groups(groups):
    with pytest.raises(KernelError):
        SharedPrefixes(groups, 4, 8, 2, "cpu")


def test_refused_heads():
    for heads in ((8, 3), (0, 1), (8, 0)):
        with pytest.raises(KernelError):
            SharedPrefixes([], 4, *heads, "cpu")
    with pytest.raises(KernelError):
        SharedPrefixes([([0, 1], 5)], 4, 256, 1, "cpu")


# ------------------------------------------------------------------------------------------------- pages with several holders
def manager(num_pages=16, page=4, max_seqs=8, needs=None):
    from rvllm_b200.cache import CacheManager
    from rvllm_b200.parts import KvCacheNeed
    return CacheManager(needs or {0: KvCacheNeed(2, 16, None), 1: KvCacheNeed(1, 16, None)}, num_pages, page, max_seqs, torch.float32, "cpu", allocate=False)


def test_a_shared_page_is_free_when_its_last_holder_gives_it_back():
    from rvllm_b200 import SchedulerError
    m = manager()
    m.admit("a"); m.append("a", 10)
    m.admit("b"); m.share("b", "a", 8)
    assert m.num_tokens("b") == 8 and m.append("b", 3) == 8
    assert m.block_table("b", 0)[:2] == m.block_table("a", 0)[:2] and m.block_table("b", 1)[2] != m.block_table("a", 1)[2]
    assert m.num_free_pages() == [12, 12]
    m.check()
    m.admit("c"); m.share("c", "b", 8)
    m.free("a")
    m.check()
    assert m.num_free_pages() == [13, 13]
    m.free("c"); m.check()
    assert m.num_free_pages() == [13, 13]
    with pytest.raises(SchedulerError, match="held by"):
        m.groups[0].pool.release([m.block_table("b", 0)[0]], "a")
    m.free("b"); m.check()
    assert m.num_free_pages() == [16, 16]


def test_a_page_twice_in_one_table_is_found():
    """A page that several requests hold is in their tables once each: not in one twice, and in no fewer than hold it."""
    from rvllm_b200 import SchedulerError
    m = manager()
    m.admit("a"); m.append("a", 12)
    m.admit("b"); m.share("b", "a", 8)
    m.check()
    for req in ("a", "b"):
        table = m.requests[req].tables[0]
        kept = list(table)
        for at in range(1, len(table)):
            table[at] = table[0]
            with pytest.raises(SchedulerError, match="twice"):
                m.check()
            table[:] = kept
    table = m.requests["b"].tables[0]
    gone = table.pop()                               # b gives it up without saying so: its holder would keep the page for good
    with pytest.raises(SchedulerError, match="holders"):
        m.check()
    table.append(gone)
    m.check()


def test_what_cannot_be_shared_is_refused():
    from rvllm_b200 import SchedulerError
    from rvllm_b200.parts import KvCacheNeed, StateNeed
    m = manager()
    m.admit("a"); m.append("a", 10); m.admit("b")
    for n in (0, 3, 12, -4):
        with pytest.raises(SchedulerError):
            m.share("b", "a", n)
    m.append("b", 1)
    with pytest.raises(SchedulerError, match="has tokens"):
        m.share("b", "a", 4)
    m.check()
    pool = m.groups[0].pool
    with pytest.raises(SchedulerError, match="not held"):
        pool.share([15], "b")
    with pytest.raises(SchedulerError, match="already"):
        pool.share([m.block_table("a", 0)[0]], "a")
    for needs in ({0: KvCacheNeed(2, 16, 20)}, {0: KvCacheNeed(2, 16, None), 1: StateNeed((4,))}, {0: KvCacheNeed(2, 16, None, chunk=8)}, {0: StateNeed((4,))}):
        w = manager(needs=needs)
        w.admit("a"); w.append("a", 8); w.admit("b")
        assert not w.can_share and w.shared_groups(["a", "b"]) == []
        with pytest.raises(SchedulerError):
            w.share("b", "a", 4)


def test_groups_that_save_the_most():
    m = manager(num_pages=400, page=4, max_seqs=20)
    m.admit("root"); m.append("root", 8)
    # two sets of four that share 100 tokens each, all of them 8; and two that share nothing
    for s in "xy":
        m.admit(s + "0"); m.share(s + "0", "root", 8); m.append(s + "0", 92 + 3)
        for i in (1, 2, 3):
            m.admit(s + str(i)); m.share(s + str(i), s + "0", 100); m.append(s + str(i), i)
    m.admit("p"); m.append("p", 9); m.admit("q"); m.append("q", 9)
    names = ["p", "x1", "y3", "x0", "q", "y0", "x3", "y2", "x2", "y1"]
    groups = {tuple(sorted(names[i] for i in ms)): t for ms, t in m.shared_groups(names)}
    assert groups == {("x0", "x1", "x2", "x3"): 100, ("y0", "y1", "y2", "y3"): 100}
    # of six that share 8 tokens, two share 8 more: the six are worth more
    m2 = manager(num_pages=100)
    m2.admit("a"); m2.append("a", 20)
    for i in range(4):
        m2.admit(i); m2.share(i, "a", 8); m2.append(i, 2)
    m2.admit("b"); m2.share("b", "a", 16); m2.append("b", 1)
    assert [(sorted(map(str, (["a", 0, 1, 2, 3, "b"][i] for i in ms))), t) for ms, t in m2.shared_groups(["a", 0, 1, 2, 3, "b"])] == \
        [(["0", "1", "2", "3", "a", "b"], 8)]
    assert m2.shared_groups(["a"]) == [] and m2.shared_groups([]) == []


@pytest.mark.parametrize("seed", range(6))
def test_groups_against_a_plain_search(seed):
    """Which pages two requests have in common, compared one by one, at lengths around those of runs that are compared at a time."""
    rng = random.Random(seed)
    m = manager(num_pages=4000, page=2, max_seqs=64)
    m.admit(0); m.append(0, 2 * rng.choice((1, 2, 3, 31, 64)) + 1)
    for i in range(1, 30):
        m.admit(i)
        donor = rng.randrange(i)
        whole = m.num_tokens(donor) // 2
        if whole and rng.random() < 0.8:
            m.share(i, donor, 2 * rng.choice((1, whole, rng.randint(1, whole))))
        m.append(i, rng.randint(1, 40))
    names = rng.sample(range(30), rng.randint(2, 30))
    common = lambda a, b: next((k for k, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))  # noqa: E731
    tables = [m.block_table(n, 0) for n in names]
    seen = set()
    for ms, tokens in m.shared_groups(names):
        assert len(ms) > 1 and not seen & set(ms)
        seen |= set(ms)
        assert tokens == 2 * min(common(tables[ms[0]], tables[i]) for i in ms[1:]) > 0
    best = max(common(a, b) for i, a in enumerate(tables) for b in tables[:i])
    assert bool(seen) == (best > 0)


def test_nothing_is_looked_for_where_no_page_is_shared(monkeypatch):
    from rvllm_b200.engine import StepEntry
    from rvllm_b200.parts import KvCacheNeed
    r = runner({0: KvCacheNeed(2, 128, None)}, torch.bfloat16)
    looked = []
    original = r.cache.shared_groups
    monkeypatch.setattr(r.cache, "shared_groups", lambda reqs: (looked.append(tuple(reqs)), original(reqs))[1])
    for i in range(3):
        r.cache.admit(i); r.cache.append(i, 64)
    entries = [StepEntry(i, [1], (0,)) for i in range(3)]
    assert r._shared_groups(entries, [64] * 3) == [] and not looked
    r.cache.admit(3); r.cache.share(3, 1, 64)
    entries.append(StepEntry(3, [1], (0,)))
    assert r._shared_groups(entries, [64] * 4) == [([1, 3], 64)] and looked == [(0, 1, 2, 3)]
    r.cache.free(1)                                  # its pages have one holder again
    assert r._shared_groups(entries[:1] + entries[2:], [64] * 3) == [] and len(looked) == 1


def test_beginnings_within_one_another():
    """1,500 requests, each of which goes on from the one before: a chain as deep as the step is wide."""
    n = 1500
    m = manager(num_pages=3 * n + 10, page=1, max_seqs=n + 1)
    m.admit(0); m.append(0, 2)
    for i in range(1, n):
        m.admit(i); m.share(i, i - 1, i); m.append(i, 2)
    groups = m.shared_groups(list(range(n)))
    assert groups and all(len(ms) > 1 for ms, _ in groups) and sorted(x for ms, _ in groups for x in ms) == sorted({x for ms, _ in groups for x in ms})
    for ms, t in groups:
        assert len({tuple(m.block_table(i, 0)[:t]) for i in ms}) == 1


def test_other_groups_need_a_capacity():
    """Without one a launch is sized for the first groups: sixteen members where two were would leave rows of a tile uncomputed."""
    wide = [(list(range(16)), 64)]
    exact = SharedPrefixes([([0, 1], 64)], 16, 16, 4, "cpu")
    before = exact.device_ints.clone()
    with pytest.raises(KernelError):
        exact.refill(wide)
    assert torch.equal(exact.device_ints, before) and exact.widest == 2
    roomy = SharedPrefixes([([0, 1], 64)], 16, 16, 4, "cpu", capacity=(2, 8))
    assert roomy.widest == 32                        # whatever the groups, every row of a tile is computed
    roomy.refill(wide)
    again = SharedPrefixes(wide, 16, 16, 4, "cpu", capacity=(2, 8))
    assert torch.equal(roomy.device_ints, again.device_ints)
    sizes = lambda p: (p.capacity, p.most_parts, p.shortest, p.longest, p.widest)  # noqa: E731
    assert sizes(roomy) == sizes(again)


def test_refused_groups_leave_a_step_as_it_was():
    """Groups that a layout refuses are refused again, and all arrays still hold the groups before."""
    step = StepPrefixes([([0, 1], 64)], 4, "cpu", 2)
    made = [step.layout(4, 2), step.layout(6, 1)]
    before = [m.device_ints.clone() for m in made]
    for bad in ([([0, 9], 64)], [([0, 1], 64), ([1, 2], 64)], [([0, 1], 8), ([2], 4), ([3], 4)], [([0, 1], -1)]):
        for _ in range(2):
            with pytest.raises(KernelError):
                step.set_groups(bad)
        assert step.groups == [([0, 1], 64)] and all(torch.equal(m.device_ints, b) for m, b in zip(made, before))
    step.set_groups([([2, 3], 128)])
    assert step.groups == [([2, 3], 128)] and made[0].own_start.tolist() == made[1].own_start.tolist() == [0, 0, 128, 128]


def test_a_step_keeps_groups_of_its_own():
    """A caller that goes on with its lists finds what it then sets in the arrays."""
    members = [0, 1]
    groups = [(members, 64)]
    step = StepPrefixes(groups, 4, "cpu", 2)
    made = step.layout(4, 2)
    members.append(2)
    step.set_groups(groups)
    assert made.own_start.tolist() == [64, 64, 64, 0]
    groups.append(([2], 8))
    groups[0] = ([3, 1], 128)
    step.set_groups(groups)
    assert made.own_start.tolist() == [0, 128, 0, 128]


# ------------------------------------------------------------------------------------------------------------- scheduling
def scheduler(num_pages=64, page=4, max_seqs=8, budget=64, chunk=None, chunked=True, share=True, max_len=256):
    from rvllm_b200.cache import CacheManager
    from rvllm_b200.engine import Scheduler
    from rvllm_b200.parts import KvCacheNeed
    cache = CacheManager({0: KvCacheNeed(1, 16, None)}, num_pages, page, max_seqs, allocate=False)
    return cache, Scheduler(cache, max_seqs, budget, max_len, chunk, chunked, (), share_prefixes=share)


def run_step(cache, sched):
    batch = sched.schedule()
    for e in batch.entries:
        cache.append(e.request.req_id, e.num_tokens)
        assert cache.num_tokens(e.request.req_id) == e.start + e.num_tokens
    done = sched.update(batch, {e.request.req_id: 1000 + 7 * hash(e.request.req_id) % 50 + len(e.request.output) for e in batch.entries if e.samples})
    cache.check()
    return batch, done


def request(rid, prompt, max_tokens=4):
    from rvllm_b200 import SamplingParams
    from rvllm_b200.engine import Request
    return Request(rid, list(prompt), SamplingParams(max_tokens=max_tokens))


def shape(batch):
    return [(e.request.req_id, e.start, e.num_tokens, e.samples) for e in batch.entries]


def test_a_request_starts_behind_what_another_has_computed():
    cache, s = scheduler()
    s.add_request(request("a", range(30)))
    run_step(cache, s)
    s.add_request(request("b", list(range(22)) + [99] * 5))
    s.add_request(request("c", range(30)))                     # the same prompt: its last token is its own
    s.add_request(request("d", [7] * 10))
    b, _ = run_step(cache, s)
    assert shape(b) == [("a", 30, 1, True), ("b", 20, 7, True), ("c", 28, 2, True), ("d", 0, 10, True)]
    assert cache.block_table("b", 0)[:5] == cache.block_table("a", 0)[:5] and cache.block_table("c", 0)[:7] == cache.block_table("a", 0)[:7]
    while s.has_unfinished():
        run_step(cache, s)
    assert cache.num_free_pages() == [64]


def test_samples_of_one_prompt_wait_for_the_first_and_others_pass():
    cache, s = scheduler(budget=16, chunk=16)
    for i in range(3):
        s.add_request(request(i, range(40)))
    s.add_request(request("x", [5] * 6))
    got = [shape(run_step(cache, s)[0]) for _ in range(4)]
    # the first is computed in portions; the others are admitted when all but 4 pages of what they share is there
    assert got[0] == [(0, 0, 16, False)] and got[1][0] == (0, 16, 16, False)
    assert any(e[0] == "x" for g in got[:4] for e in g) or any(e[0] == "x" for e in shape(run_step(cache, s)[0]))
    seen = {}
    while s.has_unfinished():
        b, _ = run_step(cache, s)
        for e in b.entries:
            seen.setdefault(e.request.req_id, e.start)
    for g in got:
        for rid, start, _, _ in g:
            seen[rid] = min(seen.get(rid, start), start)
    assert seen[1] >= 24 and seen[2] >= 24
    assert cache.num_free_pages() == [64]


def test_without_the_option_nothing_is_shared():
    cache, s = scheduler(share=False)
    for i in range(3):
        s.add_request(request(i, range(20)))
    b, _ = run_step(cache, s)
    assert shape(b) == [(0, 0, 20, True), (1, 0, 20, True), (2, 0, 20, True)]


def test_what_two_have_in_common_is_not_kept_by_address(monkeypatch):
    """Objects of requests that ended leave their addresses to others."""
    monkeypatch.setattr("rvllm_b200.engine.scheduler.id", lambda _: 1, raising=False)
    cache, s = scheduler()
    s.add_request(request("a", range(30), max_tokens=2))
    s.add_request(request("b", range(50, 80), max_tokens=20))
    run_step(cache, s)
    w = request("w", list(range(50, 74)) + [1], max_tokens=9)
    s.add_request(w)
    for _ in range(4):
        run_step(cache, s)
    assert w.shared_tokens == 24


@pytest.mark.parametrize("seed", range(8))
def test_no_page_is_lost_under_random_arrivals_and_preemption(seed):
    rng = random.Random(seed)
    cache, s = scheduler(num_pages=rng.randint(22, 40), max_seqs=6, budget=rng.choice((8, 16, 40)), chunk=rng.choice((None, 7)), max_len=80)
    stems = [[rng.randint(0, 9) for _ in range(rng.randint(4, 40))] for _ in range(3)]
    todo = [request(i, rng.choice(stems)[:rng.randint(1, 40)] + [rng.randint(0, 9) for _ in range(rng.randint(1, 6))], rng.randint(1, 30)) for i in range(20)]
    reqs, steps, shared = list(todo), 0, 0
    while todo or s.has_unfinished():
        while todo and rng.random() < 0.5:
            s.add_request(todo.pop())
        if not s.has_unfinished():
            continue
        run_step(cache, s)
        shared += sum(r.shared_tokens for r in s.running)
        steps += 1
        if rng.random() < 0.03 and s.running:
            s.abort(rng.choice(s.running).req_id)
            cache.check()
        assert steps < 3000
    assert cache.num_free_pages() == [cache.num_pages] and shared > 0
    for r in reqs:
        assert r.finish_reason == "abort" or len(r.output) == r.params.max_tokens


def test_samples_per_prompt():
    from rvllm_b200 import SamplingError, SamplingParams
    assert SamplingParams().n == 1
    with pytest.raises(SamplingError):
        SamplingParams(n=0)


@pytest.fixture
def emulated():
    import rvllm_b200.kernels as kernel_pkg
    from emulated_kernels import EmulatedKernels
    kernel_pkg.set_library(EmulatedKernels())
    yield
    kernel_pkg.set_library(None)


def test_a_request_is_one_sample(emulated):
    from rvllm_b200 import LLM, SamplingError, SamplingParams
    from model_tools import model_folder
    llm = LLM(model_folder("tiny_llama"), dtype="float32", device="cpu", block_size=8, num_blocks=32, max_model_len=64, max_num_seqs=3)
    with pytest.raises(SamplingError, match="one sample"):
        llm.add_request([1, 2, 3], SamplingParams(n=2))
    assert not llm.scheduler.has_unfinished()
    out, = llm.generate([[1, 2, 3]], SamplingParams(n=2, max_tokens=4, ignore_eos=True))
    assert [len(o.token_ids) for o in out.outputs] == [4, 4] and out.outputs[0].token_ids == out.outputs[1].token_ids


def test_samples_on_the_command_line(emulated, monkeypatch, capsys):
    import json
    from model_tools import model_folder
    from rvllm_b200 import LLM, cli
    made = []
    monkeypatch.setattr(cli, "_llm", lambda args, **kw: made.append(args) or LLM(
        args.model, dtype="float32", device="cpu", block_size=8, num_blocks=32, max_model_len=64, max_num_seqs=3, share_prefixes=args.share_prefixes))
    assert cli.main(["generate", "--model", model_folder("tiny_llama"), "--prompt-ids", "1,2,3", "--max-tokens", "4", "--n", "2", "--share-prefixes"]) == 0
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    assert made[0].share_prefixes and [x["sample"] for x in lines] == [0, 1] and lines[0]["token_ids"] == lines[1]["token_ids"]


def test_when_a_step_reads_shared_beginnings_once():
    """The rule, at the sizes of a layer of 8 key/value heads of 128 in bfloat16 (4 KB a key) and of 4 in float32."""
    from types import SimpleNamespace
    from rvllm_b200.engine.step import ModelRunner
    half = SimpleNamespace(cache=SimpleNamespace(dtype=torch.bfloat16), _key_bytes=4096)
    worth = lambda r, n, shared, own: ModelRunner._worth_sharing(r, [(list(range(n)), shared)], n * (shared + own))  # noqa: E731
    assert not worth(half, 2, 64, 5) and not worth(half, 16, 256, 16) and worth(half, 16, 512, 16) and worth(half, 64, 2048, 1024)
    assert not worth(half, 64, 512, 1024) and worth(half, 4, 8192, 100)
    full = SimpleNamespace(cache=SimpleNamespace(dtype=torch.float32), _key_bytes=4096)
    assert not worth(full, 2, 128, 5) and worth(full, 2, 256, 5) and worth(full, 64, 64, 5)


def runner(needs, dtype, page=16, num_pages=300, max_seqs=8):
    """A step function over a cache without tensors, whose device tables are taken to exist, and the kernel library's own rules."""
    from rvllm_b200.cache import CacheManager
    from rvllm_b200.engine.step import ModelRunner
    from rvllm_b200.kernels.library import CudaKernels
    cache = CacheManager(needs, num_pages, page, max_seqs, dtype, "cpu", allocate=False)
    r = ModelRunner(None, cache, CudaKernels.__new__(CudaKernels), 4096, "cpu")
    r._page_table = torch.zeros(1)
    r._worth_sharing = lambda groups, keys: True
    return r


def decoded(r, tokens=64, n=3):
    """(entries, starts) of a decode step of n requests that share their first `tokens` tokens."""
    from rvllm_b200.engine import StepEntry
    r.cache.admit(0); r.cache.append(0, tokens)
    for i in range(1, n):
        r.cache.admit(i); r.cache.share(i, 0, tokens)
    return [StepEntry(i, [1], (0,)) for i in range(n)], [r.cache.append(i, 1) for i in range(n)]


def test_heads_whose_shared_beginnings_are_read_once():
    """bfloat16 heads and pages that the tensor-core kernel does not take stay with the decode kernel that does take them."""
    from rvllm_b200.parts import KvCacheNeed
    bf, f32 = torch.bfloat16, torch.float32
    for dtype, head, page, shares in ((bf, 128, 16, True), (bf, 64, 8, True), (bf, 96, 16, False), (bf, 80, 16, False), (bf, 256, 16, False),
                                      (bf, 32, 16, False), (bf, 128, 4, False), (bf, 64, 24, False), (f32, 96, 16, True), (f32, 20, 4, True),
                                      (f32, 260, 16, False), (f32, 18, 16, False)):
        r = runner({0: KvCacheNeed(2, head, None)}, dtype, page)
        groups = r._shared_groups(*decoded(r, 96))
        assert groups == ([([0, 1, 2], 96)] if shares else []), (dtype, head, page)
    both = runner({0: KvCacheNeed(2, 96, None), 1: KvCacheNeed(1, 128, None)}, bf)
    assert both._key_bytes == 2 * 128 * 2 and both._shared_groups(*decoded(both)) == [([0, 1, 2], 64)]


def test_caches_that_no_attention_reads_once_make_no_groups():
    """A row that is key and value at once, and pages of unlike rows: the pages are shared, the steps are those of any batch."""
    from rvllm_b200.parts import KvCacheNeed
    for dtype in (torch.bfloat16, torch.float32):
        for need in (KvCacheNeed(1, 576, None, planes=1), KvCacheNeed(1, 64, None, planes=1), KvCacheNeed(2, 64, None, 2, 128)):
            r = runner({0: need}, dtype)
            assert r.cache.can_share and r._shared_groups(*decoded(r)) == []
        mixed = runner({0: KvCacheNeed(1, 128, None, planes=1), 1: KvCacheNeed(2, 64, None)}, dtype)
        assert mixed._shared_groups(*decoded(mixed)) == [([0, 1, 2], 64)]


def test_when_a_graph_reads_shared_beginnings_once():
    """A captured step, which is launched for any groups that fit it, asks for more: at 8 key/value heads of 128 in bfloat16."""
    from rvllm_b200.engine.step import ModelRunner
    from rvllm_b200.parts import KvCacheNeed

    def shares(n, tokens, graph, need=KvCacheNeed(8, 128, None)):
        r = runner({0: need}, torch.bfloat16, num_pages=2000, max_seqs=64)
        del r._worth_sharing
        assert type(r)._worth_sharing is ModelRunner._worth_sharing
        return bool(r._shared_groups(*decoded(r, tokens, n), graph=graph))
    for n, tokens, eager, graph in ((16, 256, False, False), (16, 512, True, False), (2, 8192, True, False), (8, 2048, True, True), (16, 1024, True, True),
                                    (64, 128, True, True), (32, 256, True, True)):
        assert shares(n, tokens, False) == eager and shares(n, tokens, True) == graph, (n, tokens)
    one = KvCacheNeed(1, 128, None)
    assert shares(32, 2048, True, one) and not shares(32, 1024, True, one)
    r = runner({0: KvCacheNeed(8, 128, None)}, torch.bfloat16, num_pages=2000)    # the one does not stay for the other
    del r._worth_sharing
    step = decoded(r, 8192, 2)
    assert [bool(r._shared_groups(*step, graph=g)) for g in (True, False, True, False)] == [False, True, False, True]


def test_only_graphs_are_laid_out_for_so_many_groups():
    """Of eleven prompts' samples a graph takes the eight that save the most, a step by itself all."""
    from rvllm_b200.engine import StepEntry
    from rvllm_b200.parts import KvCacheNeed
    r = runner({0: KvCacheNeed(8, 128, None)}, torch.bfloat16, num_pages=2000, max_seqs=40)
    names = []
    for g in range(11):
        r.cache.admit((g, 0)); r.cache.append((g, 0), 16 * (g + 1))
        for i in (1, 2):
            r.cache.admit((g, i)); r.cache.share((g, i), (g, 0), 16 * (g + 1))
        names += [(g, i) for i in range(3)]
    entries, starts = [StepEntry(n, [1], (0,)) for n in names], [r.cache.append(n, 1) for n in names]
    for graph, n in ((True, 8), (False, 11), (True, 8)):
        groups = r._shared_groups(entries, starts, graph=graph)
        assert [t for _, t in groups] == [16 * (g + 1) for g in range(10, 10 - n, -1)]


def test_pieces_of_the_own_keys():
    """The parts' sums stay small however many sequences there are and however long they are; a few sequences have a warp a chunk."""
    from rvllm_b200.kernels.library import CudaKernels
    k = CudaKernels.__new__(CudaKernels)
    k.num_sms = 148
    assert k._own_pieces(4, 7) == (16, 1, 1) and k._own_pieces(32, 157) == (16, 10, 80)
    assert k._own_pieces(456, 399)[:2] == (64, 7) and k._own_pieces(512, 692)[:2] == (128, 6) and k._own_pieces(2048, 2000)[:2] == (256, 8)
    for pairs in (1, 30, 500, 2048, 16384, 65536):
        for most in (1, 15, 16, 17, 300, 4000, 70000, 2 ** 20, 2 ** 31 - 1):
            piece, pieces, ctas = k._own_pieces(pairs, most)
            assert (pieces - 1) * piece < most <= pieces * piece and 1 <= ctas <= 296 and 4 * (ctas - 1) < pairs * pieces
            assert pieces <= 64 and (pieces <= 8 or pairs * pieces <= 8 * 4 * 296)
