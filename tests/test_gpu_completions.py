"""Forked completions, scores and the 8-bit cache through the engine on the device."""
import pytest
import torch

from conftest import PAGE_SIZE, TINY, random_tokens
from gpu_common import stored_dtype
from pytriton_llama_b200 import EngineConfig, SamplingParams
from pytriton_llama_b200.engine.engine import Engine, StepEntry
from pytriton_llama_b200.engine.llm import LLM

pytestmark = pytest.mark.gpu
NAMES = ["B", "D", "E", "F", "H"]


def _config(name, dtype, **more):
    opts = dict(dtype=dtype, page_size=max(16, PAGE_SIZE[name]), max_gpu_num_blocks=120, max_seq_len=512, max_num_seqs=8, seed=5)
    opts.update(more)
    return EngineConfig(**opts)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", NAMES)
def test_both_caches_hold_the_same_first_layer(model_folders, name, dtype):
    """Half a step apart, and half a rounding of the type where one of them rounds a rotated key the other way."""
    folder = model_folders(name, stored_dtype(dtype))
    seq = random_tokens(150, TINY[name]["vocab_size"], 8)
    held = []
    for bits in (None, 8):
        eng = Engine(folder, _config(name, dtype, cache_bits=bits), device="cuda:0")
        eng.step([StepEntry("a", seq[:70])])
        eng.step([StepEntry("a", seq[70:100]), StepEntry("b", seq[:3])])
        for t in seq[100:]:
            out = eng.step([StepEntry("a", [t], want=[0]), StepEntry("b", [t])])
        assert torch.isfinite(out.logits).all()
        held.append(eng.cached_kv("a", 0).double())
        eng.check_device_status()
    x = torch.cat([held[0], torch.zeros_like(held[0][:10])])
    big = x.unflatten(0, (10, 16)).abs().amax((1, 4), keepdim=True).expand(10, 16, *x.shape[1:]).flatten(0, 1)[:150]
    ulp = torch.finfo(stored_dtype(dtype)).eps
    # (an exponent may be the next one where the largest rounds up to a power of two; float32 angles' cosines differ by a few ulps)
    assert ((held[1] - held[0]).abs() <= torch.exp2(torch.floor(torch.log2(big * (1 + ulp))) - 7) + (ulp if dtype == "bfloat16" else 8 * ulp) * big).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", ["D", "E", "H"])
def test_captured_steps_give_the_same_tokens(model_folders, name, dtype):
    folder = model_folders(name, stored_dtype(dtype))
    vocab = TINY[name]["vocab_size"]
    prompts = [random_tokens(n, vocab, n) for n in (33, 5, 100, 17, 64)]
    params = SamplingParams(temperature=0.8, max_gen_len=40, top_logprobs=4, n=2)
    got = []
    for compiled in (False, True):
        for overlap in (False, True):
            llm = LLM(folder, _config(name, dtype, cache_bits=8, compiled_model=compiled, capture_mixed_steps=False, overlap_steps=overlap,
                                      max_seq_len=256, graph_context_buckets=()))
            reqs = [llm.add_request(p, params) for p in prompts]
            for _ in llm.run():
                pass
            reqs = llm._with_siblings(reqs)
            got.append([(r.output, r.logprobs, r.entropies, r.top_logprobs) for r in reqs])
            assert all(len(r.output) == 40 or r.finish_reason == "stop" for r in reqs)
            llm.engine.check_device_status()
            llm.engine.cache.check_invariants()
    assert got[0] == got[1] and got[2] == got[3]
    for one, other in zip(got[0], got[2]):          # captured: the key splits are those of the longest context, sums differ in their last bits
        same = next((i for i, (a, b) in enumerate(zip(one[0], other[0])) if a != b), len(one[0]))
        assert same > 0


@pytest.mark.parametrize("bits", [None, 8])
def test_a_forked_request_continues_as_its_parent(model_folders, bits):
    folder = model_folders("D", torch.bfloat16)
    vocab = TINY["D"]["vocab_size"]
    eng = Engine(folder, _config("D", "bfloat16", cache_bits=bits), device="cuda:0")
    eng.step([StepEntry("x", random_tokens(90, vocab, 3))])
    eng.step([StepEntry("a", random_tokens(77, vocab, 1))])
    eng.fork("a", ["b", "c"])
    rest = random_tokens(20, vocab, 2)
    for i, t in enumerate(rest):
        rows = [eng.step([StepEntry(r, [t], want=[0])]).logits for r in "ab"]
        assert torch.equal(rows[0], rows[1])
        if i == 7:
            eng.finish("x")
            assert eng.compact_cache() > 0
        if i == 11:
            eng.resize_cache(20)
            eng.resize_cache(70)
    both = eng.step([StepEntry("c", rest, want=[19])]).logits
    assert torch.isfinite(both).all()
    assert torch.equal(eng.cached_kv("a", 1), eng.cached_kv("b", 1))
    if bits is None:
        assert torch.equal(eng.cached_kv("c", 0)[:77], eng.cached_kv("a", 0)[:77])
    eng.check_device_status()


@pytest.mark.parametrize("module", ["tibepel", "lilenex", "sogalix", "podizen", "nesisun", "gepilix"])
def test_every_kind_of_state_is_forked(module):
    """States, block means and pages of other mixers: the fork goes on as its parent."""
    plain = __import__("plain_" + module)
    cfg = next(iter(plain.TINY.values()))
    vocab = cfg.get("vocab") or cfg["vocab_size"]
    eng = Engine(None, EngineConfig(dtype="float32", max_gpu_num_blocks=80, max_seq_len=300, max_num_seqs=4), device="cuda:0", model_config=cfg, random_seed=1)
    eng.step([StepEntry("x", random_tokens(40, vocab, 3))])
    eng.step([StepEntry("a", random_tokens(77, vocab, 1))])
    eng.fork("a", ["b"])
    eng.finish("x")
    eng.compact_cache()
    for t in random_tokens(30, vocab, 2):
        rows = [eng.step([StepEntry(r, [t], want=[0])]).logits for r in "ab"]
        assert torch.equal(rows[0], rows[1])
    with pytest.raises(ValueError, match="compute type"):
        Engine(None, EngineConfig(dtype="float32", max_gpu_num_blocks=8, cache_bits=8), device="cuda:0", model_config=cfg, random_seed=1)


def test_scores_and_generation_agree(model_folders):
    folder = model_folders("D", torch.float32)
    vocab = TINY["D"]["vocab_size"]
    llm = LLM(folder, _config("D", "float32", compiled_model=True))
    reqs = [llm.add_request(random_tokens(30, vocab, i), SamplingParams(temperature=0.7, max_gen_len=25, top_logprobs=3)) for i in range(3)]
    for _ in llm.run():
        pass
    scores = llm.score([r.prompt + r.output for r in reqs], top=3)
    for r, s in zip(reqs, scores):
        k = len(r.prompt) - 1
        # both logits are within 1e-4 of the model's
        assert (torch.tensor(r.logprobs) - torch.tensor(s.logprobs[k:])).abs().max() < 4e-4
        assert len(r.entropies) == len(r.output) == len(r.top_logprobs)


def test_captured_steps_after_the_cache_changed_its_size(model_folders):
    folder = model_folders("D", torch.bfloat16)
    vocab = TINY["D"]["vocab_size"]
    outs = []
    for resize in (False, True):
        llm = LLM(folder, _config("D", "bfloat16", compiled_model=True, cache_bits=8))
        reqs = [llm.add_request(random_tokens(40, vocab, i), SamplingParams(temperature=0.0, max_gen_len=60)) for i in range(4)]
        for i, _ in enumerate(llm.run()):
            if resize and i in (10, 30):
                llm.engine.resize_cache(40 if i == 10 else 100)
        outs.append([r.output for r in reqs])
        llm.engine.check_device_status()
    assert outs[0] == outs[1]


def test_command_line(model_folders, capsys):
    import cli
    folder = model_folders("D", torch.bfloat16)
    assert cli.main(["--checkpoints_dir", str(folder), "--prompt_ids", "1", "2", "3", "--max_gen_len", "5", "--cache_bits", "8", "--n", "3",
                     "--top_logprobs", "2", "--max_gpu_num_blocks", "64", "--max_seq_len", "128"]) == 0
    lines = capsys.readouterr().out.strip().splitlines()
    assert len([x for x in lines if not x.startswith("  ")]) == 3


def test_mixed_steps_are_captured_after_any_number_of_resizes(model_folders):
    """Beside logits that the caller still holds in the memory of the graphs that went."""
    eng = Engine(model_folders("D", torch.bfloat16), _config("D", "bfloat16", cache_bits=8, compiled_model=True, capture_mixed_steps=True), device="cuda:0")
    eng.GRAPH_MAX_CAPTURES = 4
    prompt, held, want = random_tokens(60, TINY["D"]["vocab_size"], 1), [], None
    for i in range(12):
        for _ in range(3):                                 # seen, captured, replayed
            held.append(eng.step([StepEntry("a", prompt, want=[59])], own_logits=False).logits)
            eng.finish("a")
            if len(held) > 1:                              # (the first was not captured: other key splits)
                want = held[-1].clone() if want is None else want
                assert torch.equal(held[-1], want)
        assert any(isinstance(k, tuple) for k in eng._graphs)
        eng.resize_cache(60 + i)
    eng.check_device_status()


@pytest.mark.parametrize("bits", [None, 8])
def test_a_resize_that_finds_no_memory_half_way(model_folders, bits):
    """The first cache entry's new pages fit, the second's do not: requests go on as if nothing had been asked for, captured steps among them."""
    folder = model_folders("D", torch.bfloat16)
    outs = []
    for resize in (False, True):
        llm = LLM(folder, _config("D", "bfloat16", compiled_model=True, cache_bits=bits))
        cache = llm.engine.cache
        reqs = [llm.add_request(random_tokens(40, TINY["D"]["vocab_size"], i), SamplingParams(temperature=0.0, max_gen_len=60)) for i in range(4)]
        for i, _ in enumerate(llm.run()):
            if resize and i in (10, 30):
                pages = 1 << 18
                one = pages * cache.groups[0].kv[0][0].nbytes
                torch.cuda.empty_cache()
                total = torch.cuda.get_device_properties(0).total_memory
                torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved(0) + 1.5 * one) / total, 0)
                try:
                    with pytest.raises(torch.OutOfMemoryError):
                        llm.engine.resize_cache(pages)
                finally:
                    torch.cuda.set_per_process_memory_fraction(1.0, 0)
                assert cache.groups[0].pool.num_pages == 120 and {t.shape[0] for t in cache.groups[0].page_tensors()} == {120}
        cache.check_invariants()
        llm.engine.check_device_status()
        outs.append([r.output for r in reqs])
    assert outs[0] == outs[1]
