"""Requests that share beginnings, through the Python entry point; and the tables that the device builds for a step."""
import random

import pytest
import torch

import plain_impl
import tufirax_tools
from model_tools import folder_for, model_folder, random_requests

pytestmark = pytest.mark.gpu

SHAPED = {"architectures": ["LlamaForCausalLM"], "hidden_size": 256, "num_hidden_layers": 2, "num_attention_heads": 8, "num_key_value_heads": 2,
          "head_dim": 64, "intermediate_size": 320, "vocab_size": 515, "max_position_embeddings": 2048, "rms_norm_eps": 1e-5,
          "rope_theta": 10000.0, "tie_word_embeddings": False, "hidden_act": "silu", "torch_dtype": "bfloat16"}


@pytest.fixture(autouse=True)
def collected():
    """Engines with their graphs are gone when a test ends, not in the middle of a later one's capture."""
    import gc
    yield
    gc.collect()


@pytest.fixture(autouse=True)
def share_little(monkeypatch):
    from rvllm_b200.engine.step import ModelRunner
    monkeypatch.setattr(ModelRunner, "_worth_sharing", lambda self, groups, keys: True)


def make(folder, dtype, **kw):
    from rvllm_b200 import LLM
    args = dict(dtype=dtype, block_size=8, num_blocks=256, max_model_len=512, max_num_seqs=16, max_num_batched_tokens=64, share_prefixes=True)
    args.update(kw)
    return LLM(folder, **args)


def counted(llm, monkeypatch):
    """How often the attention that reads a shared beginning once is launched, kernel by kernel (a replayed graph counts when it is captured)."""
    calls = []
    k = llm.engine.kernels
    original = k.shared_prefix_attention
    monkeypatch.setattr(k, "shared_prefix_attention", lambda *a, **kw: (calls.append(a[2].num_seqs), original(*a, **kw))[1])
    return calls


def stems(vocab, seed=0):
    return list(random_requests(vocab, (70, 41), seed=seed).values())


@pytest.mark.parametrize("eager", [True, False])
@pytest.mark.parametrize("name", ["tiny_llama", "shaped"])
def test_float32_tokens_do_not_depend_on_sharing(name, eager, monkeypatch):
    from rvllm_b200 import SamplingParams
    folder = folder_for(SHAPED) if name == "shaped" else model_folder(name)
    cfg, w = plain_impl.read_model_folder(folder)
    a, b = stems(cfg["vocab_size"])
    prompts = [a, a, a[:60] + [3, 4, 5], a, b, b[:40] + [1], [9, 8, 7], a[:33], b]
    llm = make(folder, "float32", enforce_eager=eager)
    if not llm.engine.cache.can_share:
        pytest.skip("this model has windows")
    calls = counted(llm, monkeypatch)
    sp = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
    outs = [o.outputs[0].token_ids for o in llm.generate(prompts, sp)]
    assert calls, "no step read a shared beginning once"
    assert outs[0] == outs[1] == outs[3] == plain_impl.greedy_generate(cfg, w, a, 12)
    assert outs[4] == outs[8] == plain_impl.greedy_generate(cfg, w, b, 12) and outs[2] == plain_impl.greedy_generate(cfg, w, prompts[2], 12)
    alone = make(folder, "float32", enforce_eager=eager, share_prefixes=False)
    assert outs == [o.outputs[0].token_ids for o in alone.generate(prompts, sp)]
    llm.engine.cache.check()
    assert not llm.engine.cache.requests and llm.engine.cache.num_free_pages() == [256] * len(llm.engine.cache.groups)
    # again, with other requests in the same graphs
    more = [b, a[:50] + [2], b[:24] + [5, 6], a, a]
    assert [o.outputs[0].token_ids for o in llm.generate(more, sp)] == [o.outputs[0].token_ids for o in alone.generate(more, sp)]


def test_samples_of_one_prompt(monkeypatch):
    from rvllm_b200 import SamplingParams
    folder = folder_for(SHAPED)
    a, b = stems(515, seed=4)
    llm = make(folder, "float32")
    out = llm.generate([a, b], [SamplingParams(temperature=0.9, seed=11, max_tokens=15, ignore_eos=True, n=6), SamplingParams(max_tokens=3)])
    assert [len(o.outputs) for o in out] == [6, 1]
    alone = make(folder, "float32", share_prefixes=False)
    want = [alone.generate([a], SamplingParams(temperature=0.9, seed=11 + i, max_tokens=15, ignore_eos=True))[0].outputs[0].token_ids for i in range(6)]
    assert [c.token_ids for c in out[0].outputs] == want and len({tuple(t) for t in want}) > 1
    seeds = llm.generate([a], SamplingParams(temperature=0.9, max_tokens=4, ignore_eos=True, n=3))[0].outputs
    assert len(seeds) == 3


def test_few_pages_preempt_requests_that_share():
    from rvllm_b200 import SamplingParams
    folder = folder_for(SHAPED)
    a, _ = stems(515, seed=2)
    prompts = [a, a, a[:30] + [1, 2], a, a[:55], a]
    sp = SamplingParams(temperature=0.7, seed=5, max_tokens=60, ignore_eos=True)
    tight = make(folder, "float32", num_blocks=34, max_num_seqs=6)
    outs = tight.generate(prompts, sp)
    assert sum(o.num_preemptions for o in outs) > 0
    roomy = make(folder, "float32", share_prefixes=False)
    assert [o.outputs[0].token_ids for o in outs] == [o.outputs[0].token_ids for o in roomy.generate(prompts, sp)]
    tight.engine.cache.check()
    assert tight.engine.cache.num_free_pages() == [34]


@pytest.mark.parametrize("eager", [True, False])
def test_bfloat16_logits_with_a_shared_beginning(eager, monkeypatch):
    """Step by step on given tokens: the logits of requests on shared pages stay within bfloat16's reach of those computed alone."""
    from rvllm_b200.engine import StepEntry
    folder = folder_for(SHAPED)
    a, _ = stems(515, seed=6)
    share, alone = (make(folder, "bfloat16", enforce_eager=eager, share_prefixes=s) for s in (True, False))
    calls = counted(share, monkeypatch)
    rng = random.Random(0)
    tails = [[rng.randrange(515) for _ in range(20 + i)] for i in range(5)]
    logits = []
    for llm in (share, alone):
        eng = llm.engine
        got = []
        eng.runner.step([StepEntry(0, a, ())])
        for i in range(1, 5):
            if llm is share:
                eng.cache.admit(i)
                eng.cache.share(i, 0, 64)
                eng.runner.step([StepEntry(i, a[64:] + tails[i][:1], ())])
            else:
                eng.runner.step([StepEntry(i, a + tails[i][:1], ())])
        for t in range(1, 15):
            entries = [StepEntry(i, [tails[i][t]], (0,)) for i in ((0, 1, 2, 3, 4) if t < 8 else (3, 0, 4))]
            got.append(eng.runner.step(entries).float().cpu())
        logits.append(torch.cat(got))
    assert calls
    x, y = logits
    assert float((x - y).abs().max()) <= 2e-2 * float(y.abs().max())


def test_an_identifier_that_is_used_again(monkeypatch):
    """Requests that share, end, and come back under the same identifiers with other beginnings: nothing of the first is kept."""
    from rvllm_b200.engine import StepEntry
    folder = folder_for(SHAPED)
    a, b = stems(515, seed=9)
    logits = []
    for share in (True, False):
        eng = make(folder, "float32", share_prefixes=share).engine
        got = []
        for stem in (a[:64], (b + a)[:64]):
            eng.runner.step([StepEntry(0, stem + [1], ())])
            for i in (1, 2):
                if share and stem == a[:64]:
                    eng.cache.admit(i); eng.cache.share(i, 0, 64)
                    eng.runner.step([StepEntry(i, [i + 5], ())])
                else:
                    eng.runner.step([StepEntry(i, (stem if i == 1 or stem == a[:64] else stem[::-1]) + [i + 5], ())])
            for t in range(3):
                got.append(eng.runner.step([StepEntry(i, [t + i], (0,)) for i in range(3)]).cpu())
            for i in range(3):
                eng.runner.finish(i)
        logits.append(torch.cat(got))
    # float32 sums in another order: a few hundred roundings of 2^-24 of values the size of the logits
    assert float((logits[0] - logits[1]).abs().max()) <= 2e-4 * float(logits[1].abs().max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_made_ahead_serve_steps_that_share(dtype, monkeypatch):
    """After `capture_graphs` no step of requests that share beginnings captures anything, at any length of what lies behind them."""
    from rvllm_b200 import SamplingParams
    llm = make(folder_for(SHAPED), dtype, num_blocks=600, max_model_len=1024, max_num_batched_tokens=1024)
    made = llm.capture_graphs()
    r = llm.engine.runner
    keys = set(r._graphs)
    assert made == len(keys) and (4, 768, 512) in keys and (4, 768, 768) in keys and (4, 768, 0) in keys and (1, 512, 512) not in keys
    assert not any(own > ctx for _, ctx, own in keys) and llm.capture_graphs() == 0
    calls = counted(llm, monkeypatch)
    replayed = []
    original = r._step_graph
    monkeypatch.setattr(r, "_step_graph", lambda e, s, b, late=None: (replayed.append(r._shared_groups(e, s, graph=True)), original(e, s, b, late))[1])
    a, _ = stems(515, seed=5)
    long = (a * 12)[:700]
    sp = SamplingParams(max_tokens=5, ignore_eos=True)
    for prompts in ([a, a, a], [long, long[:690] + [1]], [a + long[:650], a + [3], long[::-1]]):
        llm.generate(prompts, sp)
    assert sum(bool(g) for g in replayed) >= 8 and set(r._graphs) == keys
    assert not calls, "a step ran without its graph"


def test_no_garbage_is_collected_during_a_capture(monkeypatch):
    """That of an engine that is gone may hold graphs, whose end would end the capture (many are captured ahead for steps that share)."""
    import gc
    llm = make(folder_for(SHAPED), "float32", max_model_len=512)
    model, seen = llm.engine.model, []
    original = model.forward
    monkeypatch.setattr(model, "forward", lambda *a: (seen.append((torch.cuda.is_current_stream_capturing(), gc.isenabled())), original(*a))[1])
    for enabled in (True, False):
        (gc.enable if enabled else gc.disable)()
        try:
            llm.engine.runner._graphs.clear()
            assert llm.capture_graphs() > 0 and gc.isenabled() == enabled
        finally:
            gc.enable()
    assert {c for c, _ in seen} == {True, False} and not any(c and g for c, g in seen)


@pytest.mark.parametrize("eager", [True, False])
def test_layers_that_read_no_beginning_once_get_no_graphs_of_their_own(eager, monkeypatch):
    """Where no layer's attention asks for the groups of a step, later steps make none."""
    from rvllm_b200 import SamplingParams
    llm = make(folder_for(SHAPED), "float32", enforce_eager=eager)
    k, r = llm.engine.kernels, llm.engine.runner
    original = k.paged_attention

    def each_for_itself(q, cache, meta, *args, **kw):
        meta.shared = None
        return original(q, cache, meta, *args, **kw)
    monkeypatch.setattr(k, "paged_attention", each_for_itself)
    a, _ = stems(515, seed=3)
    llm.generate([a, a, a], SamplingParams(max_tokens=6, ignore_eos=True))
    assert not r._key_bytes and all(own == 0 for _, _, own in r._graphs)
    assert eager or r._graphs


# ------------------------------------------------------------------------------------------------------------ step tables
def windowed():
    return dict(plain_windows={"architectures": ["Qwen2ForCausalLM"], "hidden_size": 64, "num_hidden_layers": 4, "num_attention_heads": 4,
                               "num_key_value_heads": 2, "head_dim": 16, "intermediate_size": 96, "vocab_size": 131, "max_position_embeddings": 512,
                               "rms_norm_eps": 1e-6, "rope_theta": 10000.0, "tie_word_embeddings": True, "hidden_act": "silu",
                               "use_sliding_window": True, "sliding_window": 24, "max_window_layers": 2, "torch_dtype": "bfloat16"})["plain_windows"]


@pytest.mark.parametrize("model", ["windows", "tufirax", "llama"])
def test_tables_of_the_device_are_those_of_the_host(model):
    """Random steps - portions, decoded tokens, requests that end and whose slots are taken again - packed both ways."""
    from rvllm_b200.config import EngineConfig
    from rvllm_b200.engine import Engine, StepEntry
    folder = {"windows": lambda: folder_for(windowed()), "tufirax": lambda: tufirax_tools.write_folder(tufirax_tools.small_b(), seed=1),
              "llama": lambda: model_folder("tiny_llama")}[model]()
    eng = Engine(folder, engine_config=EngineConfig(dtype="float32", block_size=8, num_blocks=120, max_model_len=200, max_num_seqs=6,
                                                    max_num_batched_tokens=64, enforce_eager=True))
    r = eng.runner
    assert r._page_table is not None
    rng = random.Random(3)
    vocab, live, number = eng.spec.vocab_size, {}, 0
    for step in range(60):
        for rid in [x for x in live if rng.random() < 0.06 or live[x] > 150]:
            r.finish(rid); del live[rid]
        while len(live) < 6 and rng.random() < 0.6:
            live[number] = 0; number += 1
        chosen = rng.sample(sorted(live), rng.randint(1, len(live))) if live else []
        if not chosen:
            continue
        decode = rng.random() < 0.5
        entries = []
        for rid in chosen:
            n = 1 if decode else rng.choice((1, 2, 9, 30))
            entries.append(StepEntry(rid, [rng.randrange(vocab) for _ in range(n)], (n - 1,) if rng.random() < 0.8 else ()))
            live[rid] += n
        r.validate(entries)
        starts = r.reserve(entries)
        pad = 8 if decode and all(len(e.want) == 1 for e in entries) else None
        for p in (None, pad):
            table, r._page_table = r._page_table, None
            host = r.pack(entries, starts, pad_to=p)
            want = [(m.block_tables.clone(), m.slot_mapping.clone(), m.ctx_lens.clone()) for m in host.attention]
            rest = [t.clone() for t in (host.positions, host.token_seq, host.cu_seqlens, host.token_ids, host.state_slots, host.logit_rows)]
            r._page_table = table
            dev = r.pack(entries, starts, pad_to=p)
            for m, w in zip(dev.attention, want):
                for x, y in zip((m.block_tables, m.slot_mapping, m.ctx_lens), w):
                    assert torch.equal(x, y)
            for x, y in zip((dev.positions, dev.token_seq, dev.cu_seqlens, dev.token_ids, dev.state_slots, dev.logit_rows), rest):
                assert torch.equal(x, y)
        for e in entries:
            eng.cache.release_passed(e.req_id)


def test_tables_are_settled_where_kernels_follow_that_start_early(monkeypatch):
    """Steps without a graph, and the padded batch that a capture runs first, launch kernels right behind the tables; a replayed graph, and
    tokens that the host has not read, come with a boundary of their own."""
    from rvllm_b200.engine import StepEntry
    eng = make(folder_for(SHAPED), "float32", share_prefixes=False).engine
    k, seen = eng.kernels, []
    original = k.step_tables
    monkeypatch.setattr(k, "step_tables", lambda *a, **kw: (seen.append(kw["settle"]), original(*a, **kw))[1])
    step = lambda n, t=1, late=None: eng.runner.step([StepEntry(i, list(range(1, t + 1)), (t - 1,)) for i in range(n)], late_tokens=late)  # noqa: E731
    step(2, 5)
    assert seen == [True]                            # portions
    step(2)
    assert seen == [True, True, True]                # the first of its size: eagerly, then a batch of padding rows
    step(2)
    assert seen[3:] == [False]                       # replayed
    ids = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    step(2, late=(ids, [0, 1]))
    assert seen[4:] == [False]
