"""Several completions of a prompt, scores, and an 8-bit cache through the engine, with plain operators in place of the kernels."""
import pytest
import torch

import plain_llama
from conftest import FP32_TOL, PAGE_SIZE, TINY, random_tokens
from torch_ops8 import TorchOps8
from pytriton_llama_b200 import EngineConfig, SamplingParams
from pytriton_llama_b200.cache.manager import OutOfPages
from pytriton_llama_b200.engine.engine import Engine, StepEntry
from pytriton_llama_b200.engine.llm import LLM


def _llm(folder, name="A", pages=40, max_num_seqs=4, budget=24, seed=3, **more):
    page_size = more.pop("page_size", PAGE_SIZE[name])
    cfg = EngineConfig(dtype="float32", page_size=page_size, max_gpu_num_blocks=pages, max_seq_len=96, max_num_seqs=max_num_seqs,
                       max_batched_tokens=budget, seed=seed, **more)
    return LLM(folder, cfg, device="cpu", ops=TorchOps8())


@pytest.mark.parametrize("overlap", [True, False])
@pytest.mark.parametrize("pages,seqs", [(40, 4), (40, 2), (12, 4), (9, 3)])
def test_completions_are_those_of_separate_requests(model_folders, overlap, pages, seqs):
    """Whether they are forked, queue for slots or pages, or are pre-empted."""
    folder = model_folders("A")
    prompts = [random_tokens(n, 256, 50 + n) for n in (13, 7)]
    alone = _llm(folder)
    want = []
    for p in prompts:
        reqs = [alone.add_request(p, SamplingParams(temperature=0.9, max_gen_len=9, logprobs=True)) for _ in range(3)]
        for _ in alone.run():
            pass
        want += reqs
    llm = _llm(folder, pages=pages, max_num_seqs=seqs, overlap_steps=overlap)
    got = llm.generate(prompts, SamplingParams(temperature=0.9, max_gen_len=9, n=3))
    assert got == [r.output for r in want]
    assert len({tuple(x) for x in got[:3]}) > 1
    llm.engine.cache.check_invariants()
    assert llm.engine.cache.free_pages() == pages and llm.engine.cache.free_slots() == seqs


def test_a_prompt_runs_once(model_folders):
    llm = _llm(model_folders("A"), budget=64)
    llm.generate([random_tokens(40, 256, 1)], SamplingParams(temperature=1.0, max_gen_len=5, n=4))
    assert llm.engine.stats.tokens == 40 + 4 * 4


def test_stream_counts_completions(model_folders):
    llm = _llm(model_folders("A"))
    prompts, params = [random_tokens(5, 256, 1), random_tokens(9, 256, 2)], SamplingParams(temperature=0.8, max_gen_len=6, n=2)
    got = [[] for _ in range(4)]
    for events in llm.generate_stream(prompts, params):
        for i, toks, done in events:
            got[i] += toks
    assert got == _llm(model_folders("A")).generate(prompts, params)


def test_completions_of_prompts_that_cannot_run(model_folders):
    llm = _llm(model_folders("A"), pages=3)
    for prompt, why in (([], "empty_prompt"), ([1] * 96, "prompt_too_long"), ([1] * 40, "cache_too_small")):
        req = llm.add_request(prompt, SamplingParams(n=3))
        for _ in llm.run():
            pass
        assert [r.finish_reason for r in (req, *req.siblings)] == [why] * 3 and not llm.has_work()
    for bad in (dict(n=0), dict(top_logprobs=33), dict(top_logprobs=-1)):
        with pytest.raises(ValueError):
            SamplingParams(**bad)


def test_scores_of_prompts_and_of_what_is_generated(model_folders):
    folder = model_folders("A")
    cfg, w = plain_llama.load_model_folder(folder, dtype=torch.float64)
    llm = _llm(folder, budget=16)
    prompts = [random_tokens(n, 256, n) for n in (1, 2, 30, 17, 5, 9, 3)] + [[]]
    got = llm.score(prompts, top=4)
    for p, s in zip(prompts, got):
        if len(p) < 2:
            assert s.logprobs == s.entropies == s.top_logprobs == []
            continue
        full = torch.log_softmax(plain_llama.forward(cfg, w, p), -1)[:-1]
        assert torch.allclose(torch.tensor(s.logprobs).double(), full.gather(1, torch.tensor(p[1:])[:, None])[:, 0], atol=2 * FP32_TOL)
        assert torch.allclose(torch.tensor(s.entropies).double(), -(full.exp() * full).sum(-1), atol=20 * FP32_TOL)
        for row, best in zip(full, s.top_logprobs):
            v, i = row.sort(descending=True)
            assert [a for a, _ in best] == i[:4].tolist()
    assert llm.engine.cache.free_slots() == 4 and llm.engine.cache.free_pages() == 40
    # a generation reports what scoring it afterwards gives
    mixed = [SamplingParams(temperature=0.7, max_gen_len=8, top_logprobs=3), SamplingParams(temperature=0.7, max_gen_len=8, logprobs=True),
             SamplingParams(temperature=0.0, max_gen_len=8, top_logprobs=5), SamplingParams(temperature=0.7, max_gen_len=8)]
    reqs = [llm.add_request(prompts[2], p) for p in mixed]
    for _ in llm.run():
        pass
    for r, p in zip(reqs, mixed):
        assert len(r.top_logprobs) == len(r.entropies) == (len(r.output) if p.top_logprobs else 0)
        assert len(r.logprobs) == (len(r.output) if p.logprobs else 0)
        s = llm.score([r.prompt + r.output], top=5)[0]
        k = len(r.prompt) - 1
        assert torch.allclose(torch.tensor(r.logprobs), torch.tensor(s.logprobs[k:])[:len(r.logprobs)], atol=2 * FP32_TOL)
        for best, ref in zip(r.top_logprobs, s.top_logprobs[k:]):
            assert len(best) == p.top_logprobs and [a for a, _ in best] == [a for a, _ in ref][:p.top_logprobs]
    assert reqs[2].output == [b[0][0] for b in reqs[2].top_logprobs]


def test_scoring_beside_live_requests_and_without_room(model_folders):
    llm = _llm(model_folders("A"), pages=12)
    req = llm.add_request(random_tokens(20, 256, 4), SamplingParams(temperature=0.0, max_gen_len=10))
    want = _llm(model_folders("A")).generate([req.prompt], SamplingParams(temperature=0.0, max_gen_len=10))[0]
    llm.step()
    llm.score([random_tokens(12, 256, 5)])
    with pytest.raises(OutOfPages):
        llm.score([random_tokens(12, 256, 5), random_tokens(60, 256, 5)])
    for bad in ([[1, 999]], [[1] * 97]):
        with pytest.raises(ValueError):
            llm.score(bad)
    with pytest.raises(ValueError):
        llm.score([[1, 2]], top=33)
    for _ in llm.run():
        pass
    assert req.output == want and llm.engine.cache.free_pages() == 12 and llm.engine.cache.free_slots() == 4


def test_engine_fork_compact_resize_and_cached_values(model_folders):
    folder = model_folders("B")
    for bits, page_size in ((None, 8), (8, 16)):
        cfg = EngineConfig(dtype="float32", page_size=page_size, max_gpu_num_blocks=20, max_seq_len=96, max_num_seqs=4, cache_bits=bits)
        eng = Engine(folder, cfg, device="cpu", ops=TorchOps8())
        prompt, rest = random_tokens(21, 384, 1), random_tokens(6, 384, 2)
        eng.step([StepEntry("x", random_tokens(30, 384, 9))])
        eng.step([StepEntry("a", prompt)])
        held = eng.cached_kv("a")
        assert held.shape == (21, 2, 2, 32)
        eng.fork("a", ["b", "c"])
        eng.finish("x")
        assert eng.compact_cache() > 0
        assert torch.equal(eng.cached_kv("b"), held) and torch.equal(eng.cached_kv("a"), held)
        ref = eng.step([StepEntry("a", rest, want=range(6))]).logits
        eng.resize_cache(9 if bits is None else 6)
        one_by_one = torch.cat([eng.step([StepEntry("b", [t], want=[0])]).logits for t in rest])
        both = eng.step([StepEntry("c", rest, want=range(6))]).logits
        assert torch.equal(both, ref)
        if bits is None:        # (with 8 bits a portion's earlier rows see scales that its later ones raised)
            assert (one_by_one - ref).abs().max() < FP32_TOL
        assert torch.equal(eng.cached_kv("c"), eng.cached_kv("a"))
        eng.cache.check_invariants()
        with pytest.raises(OutOfPages):
            eng.resize_cache(2)
        with pytest.raises(ValueError):
            eng.resize_cache(0)
        eng.finish_all()


def test_an_8_bit_cache_holds_what_the_other_holds(model_folders):
    """The first layer's keys and values come from the same numbers in both: half a step, 2^-7 of the power of two below the largest of a block, apart."""
    folder = model_folders("B")
    seq = random_tokens(70, 384, 8)
    held, logits = [], []
    for bits in (None, 8):
        eng = Engine(folder, EngineConfig(dtype="float32", page_size=16, max_gpu_num_blocks=20, max_seq_len=96, cache_bits=bits), device="cpu", ops=TorchOps8())
        eng.step([StepEntry("a", seq[:50])])
        logits.append(eng.step([StepEntry("a", seq[50:], want=range(20))]).logits)
        held.append(eng.cached_kv("a", 0))
    x = torch.cat([held[0], torch.zeros(10, 2, 2, 32)])
    big = x.view(5, 16, 2, 2, 32).abs().amax((1, 4), keepdim=True).expand(5, 16, 2, 2, 32).reshape(80, 2, 2, 32)[:70]
    assert ((held[1] - held[0]).abs() <= torch.exp2(torch.floor(torch.log2(big)) - 7)).all()
    assert torch.isfinite(logits[1]).all() and not torch.equal(logits[0], logits[1])


def test_what_an_8_bit_cache_refuses(model_folders):
    from pytriton_llama_b200.config.registry import resolve_architecture  # noqa: F401
    import plain_tibepel
    for bad in (dict(cache_bits=4), dict(cache_bits=16), dict(cache_bits=8, page_size=24)):
        with pytest.raises(ValueError):
            EngineConfig(**bad)
    name = next(iter(plain_tibepel.TINY))
    with pytest.raises(ValueError, match="compute type"):
        Engine(None, EngineConfig(cache_bits=8, max_gpu_num_blocks=4), device="cpu", ops=TorchOps8(), model_config=plain_tibepel.TINY[name], random_seed=0)
    assert TINY["A"]["head_dim"] == 16


def test_captured_steps_go_before_the_pages_do(model_folders, monkeypatch):
    """Whether the new pages can be had or not: a captured step holds the old ones' addresses.  What is refused beforehand costs nothing."""
    cfg = EngineConfig(dtype="float32", page_size=16, max_gpu_num_blocks=10, max_seq_len=96, max_num_seqs=4, cache_bits=8)
    eng = Engine(model_folders("B"), cfg, device="cpu", ops=TorchOps8())
    eng.step([StepEntry("a", random_tokens(40, 384, 1))])
    held = eng.cached_kv("a")
    captured = {4: object(), (64, 4, 1, ()): object(), (128, 4, 1, ()): object()}
    real = torch.zeros

    def second_fails(*args, **kwargs):
        assert not eng._graphs
        calls.append(args)
        if len(calls) > 1:
            raise MemoryError
        return real(*args, **kwargs)
    for pages in (5, 30):
        eng._graphs.update(captured)
        calls = []
        with pytest.raises(OutOfPages):
            eng.resize_cache(2)
        assert len(eng._graphs) == 3
        with monkeypatch.context() as patch:
            patch.setattr(torch, "zeros", second_fails)
            with pytest.raises(MemoryError):
                eng.resize_cache(pages)
        assert not eng._graphs
        assert torch.equal(eng.cached_kv("a"), held)
        eng.step([StepEntry("a", [1], want=[0])])
        held = eng.cached_kv("a")
        eng.cache.check_invariants()


def test_steps_captured_again_after_a_resize_count_once(model_folders):
    """However often the cache changes its size, shapes do not use up the captures that an engine makes; those dropped for others still do.  The
    memory of the dropped graphs is not captured into again."""
    cfg = EngineConfig(dtype="float32", page_size=16, max_gpu_num_blocks=10, max_seq_len=96, max_num_seqs=4)
    eng = Engine(model_folders("B"), cfg, device="cpu", ops=TorchOps8())
    eng._shape_captures = 5                                # of shapes that others have driven out
    for pages in [12, 9] * 60:
        eng._graphs.update({4: object(), (64, 4, 1, ()): object(), (128, 4, 1, ()): object()})
        eng._shape_captures, eng._graph_pool = eng._shape_captures + 2, object()
        eng.resize_cache(pages)
        assert eng._shape_captures == 5 and eng._graph_pool is None
