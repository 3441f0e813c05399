"""Python entry points: token ids in, token ids out, through scheduler, step function and sampler.

``LLM`` is the engine-level interface.  ``GenerateText`` and ``GenerateStreamText`` keep the names
and the meaning of the arguments of lite_llama's classes (lite_llama/generate.py:52-61,87-95,
156-177; lite_llama/generate_stream.py:55-64,90-98,190-216): ``checkpoints_dir``,
``tokenizer_path``, ``max_seq_len``, ``max_gpu_num_blocks``, ``compiled_model``, ``device``;
``generate(prompt_tokens, max_gen_len, temperature, top_p, echo)``.  ``load_model`` and
``triton_weight`` are accepted and ignored: weights are always read from the folder's
safetensors files and there are no Triton kernels.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, Generator, Hashable, Iterable, List, Optional, Sequence, Tuple, Union

import torch

from ..config.engine import EngineConfig
from ..sampling.params import SamplingParams
from ..sampling.sampler import Sampler
from ..cache.manager import OutOfPages
from .engine import Engine, StepEntry
from .scheduler import PENDING, Request, Scheduler, StepPlan


@dataclass
class _Launched:
    """A step that runs on the device, and where its tokens will arrive on the host."""
    plan: StepPlan
    requests: List[Request]              # one per sampled row, in row order
    host: Optional[torch.Tensor] = None  # int32 [2, rows]: tokens, bit patterns of the log-probabilities
    event: object = None
    logprobs: bool = False
    scores: Optional[torch.Tensor] = None    # float32 [rows, 1 + 2 k]: ``Sampler.sample_device_scored``


@dataclass
class PromptScores:
    """How a model rates a prompt: entry i is about token i + 1 after the tokens before it."""
    logprobs: List[float] = field(default_factory=list)
    entropies: List[float] = field(default_factory=list)              # of the distribution that the token comes from, in nats
    top_logprobs: List[List[Tuple[int, float]]] = field(default_factory=list)   # [(token, log-probability)], best first, where asked for


class LLM:
    def __init__(self, model_dir, config: Optional[EngineConfig] = None, device="cuda:0", ops=None, **engine_options):
        """``engine_options`` go to ``Engine`` (``model_config`` and ``random_seed`` for random weights)."""
        self.engine = Engine(model_dir, config, device=device, ops=ops, **engine_options)
        cfg = self.engine.config
        self.scheduler = Scheduler(self.engine.cache, cfg.max_num_seqs, cfg.max_batched_tokens,
                                   cfg.max_seq_len, eos_token_ids=self.engine.eos_token_ids)
        self.sampler = Sampler(self.engine.ops, self.engine.device, seed=cfg.seed)
        self._next_id = 0
        self._rows: Dict[Hashable, int] = {}     # request -> its row among the tokens sampled by the last launched step
        self._turn = 0
        self._staging = []
        if self.engine.device.type == "cuda":
            # where sampled tokens arrive on the host; a buffer is read before the launch after next reuses it
            self._staging = [(torch.empty((2, cfg.max_num_seqs), dtype=torch.int32, pin_memory=True), torch.cuda.Event())
                             for _ in range(3)]

    # ------------------------------------------------------------------ requests
    def add_request(self, prompt: Sequence[int], params: Optional[SamplingParams] = None,
                    request_id: Optional[Hashable] = None) -> Request:
        if request_id is None:
            request_id = f"req-{self._next_id}"
            self._next_id += 1
        prompt = [int(t) for t in prompt]
        vocab = self.engine.vocab_size
        if any(t < 0 or t >= vocab for t in prompt):
            raise ValueError(f"the prompt has a token outside the vocabulary of {vocab}")
        return self.scheduler.add(request_id, prompt, params)

    def has_work(self) -> bool:
        return self.scheduler.has_work()

    def step(self) -> Tuple[Dict[Hashable, int], List[Request]]:
        """Runs one scheduled step and reads its tokens.  Returns (request id -> new token, requests
        that finished)."""
        launched = self._launch()
        if launched is None:
            if self.scheduler.has_work():
                raise RuntimeError("the scheduler found nothing to run although requests are pending")
            return {}, []
        return self._collect(launched)

    def run(self) -> Generator[Tuple[Dict[Hashable, int], List[Request]], None, None]:
        """Steps until no request is left, yielding what ``step`` returns for every step.  With
        ``overlap_steps`` the next step is planned and launched before the tokens of the last one are
        read: a request that goes on takes its token on the device (``StepEntry.from_row``), so the
        host's work runs beside the device's.  The tokens are the same either way; a request that a
        stop token ends has by then run one step more, whose token is dropped."""
        overlap = self.engine.config.overlap_steps
        waiting_for: Optional[_Launched] = None
        while waiting_for is not None or self.scheduler.has_work():
            launched = self._launch()
            if launched is None and waiting_for is None:
                raise RuntimeError("the scheduler found nothing to run although requests are pending")
            if waiting_for is not None:
                yield self._collect(waiting_for)
                waiting_for = None
            if launched is not None and not overlap:
                yield self._collect(launched)
            else:
                waiting_for = launched

    def _launch(self) -> Optional[_Launched]:
        plan = self.scheduler.schedule()
        if not plan.portions:
            return _Launched(plan, []) if plan.finished else None
        entries = []
        for p in plan.portions:
            req = p.request
            if req.output and req.output[-1] == PENDING and p.start + p.length == len(req.prompt) + len(req.output):
                if p.length != 1:
                    raise RuntimeError(f"request {req.id!r}: a token that has not been read yet lies inside a longer portion")
                entries.append(StepEntry(req.id, [0], [0], from_row=self._rows[req.id]))
            else:
                entries.append(StepEntry(req.id, req.tokens(p.start, p.length), [p.length - 1] if p.sample else []))
        # the plan was checked against the cache and the tokens at intake; the logits are sampled from at once
        out = self.engine.step(entries, validate=False, own_logits=False)
        logits = out.logits
        sampling = sum(p.sample for p in plan.portions)
        forked = self.scheduler.fork(plan, self.engine.fork) if any(p.sample and p.request.to_fork for p in plan.portions) else []
        reqs = [p.request for p in plan.portions if p.sample]
        if forked:        # further completions of a prompt draw their first token from its last logits
            row = {r.id: i for i, r in enumerate(reqs[:sampling])}
            logits = logits.index_select(0, torch.tensor([*range(sampling), *(row[parent.id] for _, parent in forked)], device=logits.device))
        launched = _Launched(plan, reqs)
        if reqs:
            n = len(reqs)
            tokens, lp, scores = self.sampler.sample_device_scored(logits, [r.params for r in reqs], [r.number for r in reqs],
                                                                   [len(r.output) for r in reqs], out=self.engine.sampled[:n])
            launched.logprobs = lp is not None
            if self.engine.device.type == "cuda":
                launched.host, launched.event = self._staging[self._turn % len(self._staging)]
                self._turn += 1
                launched.host[0, :n].copy_(tokens, non_blocking=True)
                if lp is not None:
                    launched.host[1, :n].view(torch.float32).copy_(lp, non_blocking=True)
                if scores is not None:
                    launched.scores = torch.empty(scores.shape, dtype=torch.float32, pin_memory=True)
                    launched.scores.copy_(scores, non_blocking=True)
                launched.event.record(torch.cuda.current_stream(self.engine.device))
            else:
                launched.host = torch.stack([tokens.cpu(), (lp if lp is not None else torch.zeros(n)).cpu().view(torch.int32)])
                launched.scores = scores
        self._rows = {r.id: i for i, r in enumerate(reqs)}
        self.scheduler.advance(plan)
        return launched

    def _collect(self, launched: _Launched) -> Tuple[Dict[Hashable, int], List[Request]]:
        finished = list(launched.plan.finished)
        reqs = launched.requests
        if not reqs:
            return {}, finished + self.scheduler.resolve(launched.plan, {})[1]
        if launched.event is not None:
            launched.event.synchronize()
        n = len(reqs)
        tokens = launched.host[0, :n].tolist()
        sampled = {r.id: t for r, t in zip(reqs, tokens)}
        logprobs = None
        if launched.logprobs:
            values = launched.host[1, :n].view(torch.float32).tolist()
            logprobs = {r.id: (v if r.params.logprobs else None) for r, v in zip(reqs, values)}
        scores = None
        if launched.scores is not None:
            rows = self.sampler.read_scores(launched.scores, [r.params for r in reqs])
            scores = {r.id: s for r, s in zip(reqs, rows) if s is not None}
        accepted, done = self.scheduler.resolve(launched.plan, sampled, logprobs, scores)
        return accepted, finished + done

    # ------------------------------------------------------------------ whole runs
    def generate(self, prompt_tokens: Sequence[Sequence[int]],
                 params: Union[None, SamplingParams, Sequence[SamplingParams]] = None) -> List[List[int]]:
        """Generated token ids of every prompt (without the prompt), in the order given; with ``SamplingParams.n`` above 1 a
        prompt's completions stand next to each other."""
        plist = self._params_list(params, len(prompt_tokens))
        reqs = self._with_siblings([self.add_request(p, sp) for p, sp in zip(prompt_tokens, plist)])
        for _ in self.run():
            pass
        self.engine.check_device_status()
        return [list(r.output) for r in reqs]

    @staticmethod
    def _with_siblings(reqs: Sequence[Request]) -> List[Request]:
        return [x for r in reqs for x in (r, *r.siblings)]

    def score(self, prompt_tokens: Sequence[Sequence[int]], top: int = 0) -> List[PromptScores]:
        """Rates prompts: the log-probability of every token but the first after those before it, the entropy of the
        distribution it comes from, and with ``top`` (up to 32) that many of the most likely tokens in its place.  Prompts take
        pages beside the requests that are live, and give them back."""
        eng, cfg = self.engine, self.engine.config
        if not 0 <= top <= 32:
            raise ValueError("top must be in 0..32")
        prompts = [[int(t) for t in p] for p in prompt_tokens]
        for p in prompts:
            if any(t < 0 or t >= eng.vocab_size for t in p):
                raise ValueError(f"a prompt has a token outside the vocabulary of {eng.vocab_size}")
            if len(p) > cfg.max_seq_len:
                raise ValueError(f"a prompt of {len(p)} tokens; max_seq_len is {cfg.max_seq_len}")
        out = [PromptScores() for _ in prompts]
        room = max(1, min(cfg.max_batched_tokens, (1 << 28) // eng.vocab_size))       # rows of logits at once: up to 1 GiB of them
        todo = [(i, 0) for i, p in enumerate(prompts) if len(p) > 1]                  # (prompt, tokens of it that have run)
        live: List[Hashable] = []
        try:
            while todo:
                entries, plan = [], []
                left = room
                for i, start in todo:
                    n = min(left, len(prompts[i]) - 1 - start)
                    key = ("score", id(out), i)
                    asks = [(e.request, len(e.tokens)) for e in entries] + [(key, n)]
                    if n <= 0 or not eng.cache.can_append(asks):
                        break
                    entries.append(StepEntry(key, prompts[i][start:start + n], list(range(n))))
                    plan.append((i, start, n))
                    left -= n
                if not entries:
                    raise OutOfPages("the cache has no room for a prompt's portion beside what is live")
                live = list({*live, *(e.request for e in entries)})
                logits = eng.step(entries, own_logits=False).logits
                nxt = torch.tensor([t for i, s, n in plan for t in prompts[i][s + 1:s + n + 1]], dtype=torch.int32, device=logits.device)
                lp, entropy, best, ids = (t.tolist() for t in eng.ops.token_scores(logits, nxt, top))
                at = 0
                for i, s, n in plan:
                    out[i].logprobs += lp[at:at + n]
                    out[i].entropies += entropy[at:at + n]
                    if top:
                        out[i].top_logprobs += [list(zip(a, b)) for a, b in zip(ids[at:at + n], best[at:at + n])]
                    at += n
                ran = {i: s + n for i, s, n in plan}
                for i, s in list(ran.items()):
                    if s == len(prompts[i]) - 1:
                        eng.finish(("score", id(out), i))
                        live.remove(("score", id(out), i))
                todo = [(i, ran.get(i, s)) for i, s in todo if ran.get(i, s) < len(prompts[i]) - 1]
        finally:
            for key in live:
                eng.finish(key)
        eng.check_device_status()
        return out

    def generate_stream(self, prompt_tokens: Sequence[Sequence[int]],
                        params: Union[None, SamplingParams, Sequence[SamplingParams]] = None
                        ) -> Generator[List[Tuple[int, List[int], bool]], None, None]:
        """Yields, after every step that produced tokens, a list of (prompt index, new token ids,
        finished); with ``SamplingParams.n`` above 1 the index counts completions, in ``generate``'s order."""
        plist = self._params_list(params, len(prompt_tokens))
        reqs = self._with_siblings([self.add_request(p, sp) for p, sp in zip(prompt_tokens, plist)])
        index = {r.id: i for i, r in enumerate(reqs)}
        early = [(index[r.id], [], True) for r in reqs if r.status == "finished"]
        if early:
            yield early
        for sampled, finished in self.run():
            done = {r.id for r in finished}
            events = [(index[rid], [tok], rid in done) for rid, tok in sampled.items() if rid in index]
            events += [(index[r.id], [], True) for r in finished if r.id in index and r.id not in sampled]
            if events:
                yield sorted(events)

    @staticmethod
    def _params_list(params, n: int) -> List[SamplingParams]:
        if params is None:
            return [SamplingParams() for _ in range(n)]
        if isinstance(params, SamplingParams):
            return [params] * n
        if len(params) != n:
            raise ValueError(f"{len(params)} sampling settings for {n} prompts")
        return list(params)


def _engine_config(max_seq_len, max_gpu_num_blocks, compiled_model, dtype, **extra) -> EngineConfig:
    return EngineConfig(dtype=dtype, max_seq_len=max_seq_len, max_gpu_num_blocks=max_gpu_num_blocks,
                        compiled_model=compiled_model, **extra)


class _TextMixin:
    tokenizer = None

    def load_tokenizer(self, tokenizer_path):
        """A Hugging Face tokenizer for the text entry points (lite_llama/generate.py:78-85); the
        token-id entry points need none."""
        if tokenizer_path is None:
            return None
        from transformers import AutoTokenizer
        return AutoTokenizer.from_pretrained(tokenizer_path, use_fast=True)

    def _need_tokenizer(self):
        if self.tokenizer is None:
            raise RuntimeError("text entry points need tokenizer_path; use generate() with token ids otherwise")
        return self.tokenizer


class GenerateText(_TextMixin):
    """lite_llama/generate.py:47-206 with a continuous-batching engine underneath."""

    def __init__(self, checkpoints_dir: str, tokenizer_path: Optional[str] = None, max_seq_len: int = 1024,
                 max_gpu_num_blocks=None, load_model: bool = True, triton_weight: bool = True,
                 compiled_model: bool = False, device: str = "cuda", dtype="bfloat16", **engine_options):
        dev = "cuda:0" if device == "cuda" else device
        self.llm = LLM(checkpoints_dir, _engine_config(max_seq_len, max_gpu_num_blocks, compiled_model, dtype,
                                                       **engine_options), device=dev)
        self.model_config = self.llm.engine.model_config
        self.tokenizer = self.load_tokenizer(tokenizer_path)
        self.device = dev

    def generate(self, prompt_tokens: List[List[int]], max_gen_len: Optional[int], temperature: float = 0.6,
                 top_p: float = 0.9, echo: bool = False, logprobs: bool = False, n: int = 1):
        """Token ids generated for each prompt, cut before the first end-of-sequence token
        (lite_llama/generate.py:192-204); with ``echo`` the prompt is put in front.  With ``logprobs``
        the result is (tokens, log-probabilities of the generated tokens), as in
        lite_llama/generete_with_probs.py:87-96,154-165.  ``n`` completions of a prompt stand next to each other."""
        params = SamplingParams(temperature=temperature, top_p=top_p, max_gen_len=max_gen_len, logprobs=logprobs, n=n)
        reqs = self.llm._with_siblings([self.llm.add_request(p, params) for p in prompt_tokens])
        prompt_tokens = [r.prompt for r in reqs]
        for _ in self.llm.run():
            pass
        self.llm.engine.check_device_status()
        eos = self.llm.engine.eos_token_ids
        toks = [_trim(p, r.output, echo, eos) for p, r in zip(prompt_tokens, reqs)]
        if not logprobs:
            return toks
        kept = [len(_trim(p, r.output, False, eos)) for p, r in zip(prompt_tokens, reqs)]
        return toks, [r.logprobs[:n] for r, n in zip(reqs, kept)]

    def text_completion(self, prompts: List[str], temperature: float = 0.6, top_p: float = 0.9,
                        max_gen_len: Optional[int] = None, echo: bool = False) -> List[str]:
        tok = self._need_tokenizer()
        ids = [tok.encode(p, add_special_tokens=True) for p in prompts]
        outs = self.generate(ids, max_gen_len, temperature, top_p, echo)
        return [tok.decode(o, skip_special_tokens=True) for o in outs]


class GenerateStreamText(_TextMixin):
    """lite_llama/generate_stream.py:51-216: the same, yielding as tokens arrive."""

    def __init__(self, checkpoints_dir: str, tokenizer_path: Optional[str] = None, max_gpu_num_blocks=None,
                 max_seq_len: int = 1024, load_model: bool = True, triton_weight: bool = True,
                 compiled_model: bool = False, device: str = "cuda", dtype="bfloat16", **engine_options):
        dev = "cuda:0" if device == "cuda" else device
        self.llm = LLM(checkpoints_dir, _engine_config(max_seq_len, max_gpu_num_blocks, compiled_model, dtype,
                                                       **engine_options), device=dev)
        self.model_config = self.llm.engine.model_config
        self.tokenizer = self.load_tokenizer(tokenizer_path)
        self.device = dev

    def generate_stream(self, prompt_tokens: List[List[int]], max_gen_len: Optional[int],
                        temperature: float = 0.6, top_p: float = 0.9, echo: bool = False
                        ) -> Generator[List[List[int]], None, None]:
        """Yields, per step, the new token ids of every prompt (an empty list where a prompt got
        none); with ``echo`` the first yield of a prompt starts with the prompt itself."""
        params = SamplingParams(temperature=temperature, top_p=top_p, max_gen_len=max_gen_len)
        eos = set(self.llm.engine.eos_token_ids)
        pending_echo = [echo] * len(prompt_tokens)
        for events in self.llm.generate_stream(prompt_tokens, params):
            batch: List[List[int]] = [[] for _ in prompt_tokens]
            for i, toks, done in events:
                new = [t for t in toks if t not in eos]
                if pending_echo[i] and (new or done):
                    new = list(prompt_tokens[i]) + new
                    pending_echo[i] = False
                batch[i] = new
            yield batch

    def text_completion_stream(self, prompts: List[str], temperature: float = 0.6, top_p: float = 0.9,
                               max_gen_len: Optional[int] = None, echo: bool = False):
        """Yields the list of {'generation': text so far, 'tokens': ids so far} after every step
        (lite_llama/generate_stream.py:190-216)."""
        tok = self._need_tokenizer()
        ids = [tok.encode(p, add_special_tokens=True) for p in prompts]
        completions = [{"generation": "", "tokens": []} for _ in prompts]
        for batch in self.generate_stream(ids, max_gen_len, temperature, top_p, echo):
            for i, new in enumerate(batch):
                if new:
                    completions[i]["tokens"] = completions[i]["tokens"] + new
                    completions[i]["generation"] = tok.decode(completions[i]["tokens"], skip_special_tokens=True)
            yield [dict(c) for c in completions]


def _trim(prompt: Sequence[int], output: Sequence[int], echo: bool, eos: Iterable[int]) -> List[int]:
    eos = set(eos)
    cut = list(output)
    for i, t in enumerate(cut):
        if t in eos:
            cut = cut[:i]
            break
    return (list(prompt) + cut) if echo else cut
