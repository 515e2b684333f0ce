"""The single-request loop: a prompt goes in, tokens come out one by one.

As the reference's `generate()` (src/runtime/generator.cpp:10-78): all prompt tokens but the
last run through the step function without logits (in portions of at most `prefill_rows`); the
last prompt token and every later token run singly and return the logits from which the next
token is sampled.  Where the runner can take a step's token from the device (and the sampler draws
there), the next step is put in the queue before the host has read the token, so the device does
not wait for the host between tokens; an end token then costs one step whose result nobody sees.  `max_positions` bounds prompt plus generated tokens (0 = the context length).
An end token is kept as the last generated token and stops the loop.
"""
from __future__ import annotations

import time
from dataclasses import dataclass, field
from typing import Callable, Iterable, List, Optional, Sequence

from ..cache.pages import OutOfPages
from ..sampling import Sampler, SamplerConfig, kept_drafts, sample_rows_on_device, verify_rows
from .runner import Runner, StepEntry


@dataclass
class GenerateResult:
    prompt_tokens: List[int]
    generated_tokens: List[int] = field(default_factory=list)
    stopped_by_end_token: bool = False
    prefill_ms: float = 0.0          # the prompt, including the sampling of the first new token
    decode_ms: float = 0.0
    decode_steps: int = 0
    drafted_tokens: int = 0          # tokens that a drafter proposed, and how many of the generated ones are such
    kept_tokens: int = 0


def generate(runner: Runner, sampler: Sampler, prompt_tokens: Sequence[int], max_positions: int = 0,
             end_tokens: Iterable[int] = (), on_token: Optional[Callable[[int], None]] = None,
             prefill_rows: Optional[int] = None, request="generate", sample=None) -> GenerateResult:
    """`sample(logits_row, sampler) -> token` replaces the sampler's own device sampling (tests without a GPU use it)."""
    prompt = [int(t) for t in prompt_tokens]
    if not prompt:
        raise ValueError("generate: prompt has no tokens")
    context = runner.max_positions
    if len(prompt) > context:
        raise ValueError(f"generate: prompt of {len(prompt)} tokens does not fit in the context length {context}")
    steps = context if max_positions <= 0 else min(max_positions, context)
    end_tokens = set(int(t) for t in end_tokens)
    chunk = min(prefill_rows or runner.max_rows, runner.max_rows)
    result = GenerateResult(prompt_tokens=prompt)

    runner.open(request)
    try:
        pos = 0
        batched = min(len(prompt) - 1, steps)
        t_start = t_first = time.perf_counter()
        while pos < batched:
            n = min(chunk, batched - pos)
            runner.step([StepEntry(request, prompt[pos:pos + n], ())])
            pos += n
        token = prompt[pos] if pos < len(prompt) else None
        ahead = sample is None and pos < steps and getattr(runner, "can_step_from_device", False) and runner.model.device.type == "cuda"

        def took(nxt) -> bool:
            """Books for one generated token; False when it ends the request."""
            nonlocal t_first
            result.generated_tokens.append(nxt)
            if len(result.generated_tokens) == 1:
                t_first = time.perf_counter()
                result.prefill_ms = (t_first - t_start) * 1e3
            else:
                result.decode_steps += 1
            if nxt in end_tokens:
                result.stopped_by_end_token = True
                return False
            if on_token is not None:
                on_token(nxt)
            return True

        if ahead:
            import torch
            landing, landed = torch.empty(1, dtype=torch.int32, pin_memory=True), torch.cuda.Event()
            logits = runner.step([StepEntry(request, [token], (0,))])
            while True:
                on_device = sample_rows_on_device(logits, [sampler])
                landing.copy_(on_device, non_blocking=True)
                landed.record()
                pos += 1
                if pos < steps:                               # the next step is queued before the host knows its token
                    logits = runner.step_from_device([request], on_device)
                landed.synchronize()
                if not took(int(landing[0])) or pos >= steps:
                    break
        else:
            while pos < steps:
                logits = runner.step([StepEntry(request, [token], (0,))])
                nxt = sampler.sample(logits[0]) if sample is None else sample(logits[0], sampler)     # the token reaches the host: the step has finished
                pos += 1
                if not took(nxt):
                    break
                token = nxt
        if result.generated_tokens:
            result.decode_ms = (time.perf_counter() - t_first) * 1e3
    finally:
        runner.close(request)
    return result


def generate_with_drafts(runner: Runner, drafter: Runner, sampler: Sampler, prompt_tokens: Sequence[int], n_drafts: int = 4, max_positions: int = 0,
                         end_tokens: Iterable[int] = (), on_token: Optional[Callable[[int], None]] = None, prefill_rows: Optional[int] = None, request="generate",
                         draft=None, judge=None) -> GenerateResult:
    """`generate` with a second, cheaper model of the same vocabulary that runs ahead: `drafter` proposes up to `n_drafts` tokens one by one, a single step of `runner`
    brings the logits at all their places, and of the proposals as many stay as leave the sequence distributed as the target's own
    (`sampling.verify_rows`; a greedy sampler's tokens are `generate`'s, and so are those of one with top-k or top-p, whose proposals stay where they are what its own draw gives:
    all but for the rounding of bfloat16 products, which add up in another order for several rows than for one).
    What was fed beyond is cut off again, so neither model may keep a state or give pages back behind a window.  Both lie on one device.
    The drafter draws at the sampler's settings from numbers of its own.  draft(logits, sampler) -> token and judge(logits, drafts, sampler, draft_logits) -> new tokens replace the device's
    (tests without a GPU use them)."""
    import torch
    prompt = [int(t) for t in prompt_tokens]
    if not prompt:
        raise ValueError("generate: prompt has no tokens")
    if n_drafts < 1 or n_drafts > 64:
        raise ValueError(f"generate: 1 to 64 drafts can be judged at once, not {n_drafts}")
    vocab = runner.model.spec.vocab_size
    if drafter is runner or drafter.model.spec.vocab_size != vocab:
        raise ValueError("generate: the drafter must be another runner whose model has the same vocabulary")
    places = [torch.device(getattr(r.model, "device", "cpu")) for r in (runner, drafter)]
    if places[0] != places[1]:
        raise ValueError(f"generate: the target lies on {places[0]} and the drafter on {places[1]}; drafts are judged where both models' logits lie")
    for r, what in ((runner, "target"), (drafter, "drafter")):
        if not r.cache.rewinds:
            raise ValueError(f"generate: the {what} keeps a state or gives pages back; drafts that fall could not be taken back")
        if len(prompt) > r.max_positions:
            raise ValueError(f"generate: prompt of {len(prompt)} tokens does not fit in the context length {r.max_positions} of the {what}")
    context = runner.max_positions
    steps = context if max_positions <= 0 else min(max_positions, context)
    end_tokens = set(int(t) for t in end_tokens)
    config = sampler.config
    own = Sampler(SamplerConfig(config.temperature, config.top_k, config.top_p, config.seed ^ 0x6472616674), vocab)
    filtered = sampler.kind == "filtered"
    most = min(n_drafts, runner.max_rows - 1)
    result = GenerateResult(prompt_tokens=prompt)
    tokens = list(prompt)                                     # all that is known; runner holds tokens[:pos]

    def feed(r, upto):
        while r.cache.length(request) < upto:
            at = r.cache.length(request)
            r.step([StepEntry(request, tokens[at:min(at + min(prefill_rows or r.max_rows, r.max_rows), upto)], ())])

    runner.open(request)
    try:
        drafter.open(request)
        try:
            pos = min(len(prompt) - 1, steps)
            t_start = t_first = time.perf_counter()
            feed(runner, pos)
            proposals = torch.zeros((1, max(most, 1)), dtype=torch.int32, device=getattr(drafter.model, "device", "cpu"))
            rows = None
            while pos < steps:
                k, made = max(0, min(most, steps - pos - 1, drafter.max_positions - pos)), 0
                if k:
                    try:
                        # what the drafter has not seen (the last token, and the one before where all of its proposals stayed), then one proposal after the other
                        feed(drafter, pos)
                        logits = drafter.step([StepEntry(request, [tokens[pos]], (0,))])
                        if rows is None and not filtered and not sampler.config.greedy:
                            rows = torch.empty((1, most, vocab), dtype=torch.float32, device=logits.device)
                        while True:
                            if rows is not None:
                                rows[0, made].copy_(logits[0])
                            token = sample_rows_on_device(logits, [own]) if draft is None else torch.tensor([draft(logits[0], own)], dtype=torch.int32)
                            proposals[0, made:made + 1].copy_(token)
                            made += 1
                            if made == k:
                                break
                            if getattr(drafter, "can_step_from_device", False):           # (the host need not know the proposal to have the next one made)
                                logits = drafter.step_from_device([request], token)
                            else:
                                logits = drafter.step([StepEntry(request, [int(token[0])], (0,))])
                    except OutOfPages:                        # what has been proposed so far is judged
                        pass
                k, drafts = made, proposals[0, :made].tolist()
                try:
                    logits = runner.step([StepEntry(request, [tokens[pos]] + drafts, tuple(range(k + 1)))])
                except OutOfPages:
                    if not k:
                        raise
                    k, drafts = 0, []                         # the last pages are the target's own
                    logits = runner.step([StepEntry(request, [tokens[pos]], (0,))])
                beside = rows[:, :k] if rows is not None and k else None
                if judge is not None:
                    new = judge(logits, drafts, sampler, beside)
                elif filtered:
                    new = kept_drafts(logits, drafts, sampler)
                else:
                    new = verify_rows(logits, proposals[:, :k].contiguous(), [sampler], beside)[0]
                result.drafted_tokens += k
                if not result.generated_tokens:
                    t_first = time.perf_counter()
                    result.prefill_ms = (t_first - t_start) * 1e3
                else:
                    result.decode_steps += 1
                pos += len(new)
                runner.truncate(request, pos)
                drafter.truncate(request, min(drafter.cache.length(request), pos))
                for i, token in enumerate(new):
                    tokens.append(int(token))
                    result.generated_tokens.append(int(token))
                    result.kept_tokens += i + 1 < len(new)                # (the last is the target's own; drafts behind an end token are not taken)
                    if token in end_tokens:
                        result.stopped_by_end_token = True
                        break
                    if on_token is not None:
                        on_token(int(token))
                if result.stopped_by_end_token:
                    break
            if result.generated_tokens:
                result.decode_ms = (time.perf_counter() - t_first) * 1e3
        finally:
            drafter.close(request)
    finally:
        runner.close(request)
    return result
