"""Generation with a drafter, without a GPU: stand-in step functions over the real cache manager, drafts judged by the plain statement of the rules."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import plain_drafts
from geneinfer_amd.cache import CacheManager, OutOfPages, PagedKvNeed, StateNeed
from geneinfer_amd.engine import generate, generate_with_drafts
from geneinfer_amd.sampling import Sampler, SamplerConfig, kept_drafts, verify_rows_on_device
from test_scheduler import VOCAB, FakeRunner, host_sample_row


class Runner(FakeRunner):
    """With rewinding, and logits of its own (`twist`) on top of those that depend on the request's tokens."""

    def __init__(self, twist=0.0, **kw):
        super().__init__(**kw)
        self.twist = twist

    def truncate(self, r, length):
        self.cache.truncate(r, length)
        del self.fed[r][length:]

    def step(self, entries):
        logits = super().step(entries)
        if logits is not None and self.twist:
            logits = logits + self.twist * torch.from_numpy(np.random.default_rng(len(self.log)).standard_normal(tuple(logits.shape)).astype(np.float32))
        return logits


def judge(logits, drafts, sampler, draft_logits):
    if sampler.kind == "filtered":
        return kept_drafts(logits, drafts, sampler, sample=lambda rows, samplers: [host_sample_row(row, s) for row, s in zip(rows, samplers)])
    k = len(drafts)
    uniform = np.zeros((1, k + 1), np.float32)
    if not sampler.config.greedy:
        uniform[0] = [sampler.next_uniform() for _ in range(k + 1)]
    tokens, counts = plain_drafts.verify(logits.numpy(), np.asarray([drafts], np.int32).reshape(1, k), [sampler.temperature], uniform,
                                         None if draft_logits is None else draft_logits.numpy())
    return tokens[0, :counts[0]].tolist()


def run(target, drafter, config, prompt, n_drafts=4, limit=0, end=(), **kw):
    return generate_with_drafts(target, drafter, Sampler(config, VOCAB), prompt, n_drafts, limit, end, draft=host_sample_row, judge=judge, **kw)


PROMPT = [3, 41, 7, 7, 12]


@pytest.mark.parametrize("config", [SamplerConfig(0.0), SamplerConfig(0.9, top_k=6, seed=4), SamplerConfig(0.7, top_p=0.8, seed=5), SamplerConfig(1.1, top_k=9, top_p=0.9, seed=6)])
@pytest.mark.parametrize("twist,n_drafts", [(0.0, 1), (0.0, 4), (0.6, 3), (3.0, 5)])
def test_greedy_and_filtered_tokens_are_those_without_drafts(config, twist, n_drafts):
    for limit in (0, len(PROMPT), len(PROMPT) + 1, len(PROMPT) + 13, 2):
        want = generate(Runner(), Sampler(config, VOCAB), PROMPT, limit, sample=host_sample_row)
        target, drafter = Runner(), Runner(twist)
        got = run(target, drafter, config, PROMPT, n_drafts, limit)
        assert got.generated_tokens == want.generated_tokens
        assert got.kept_tokens <= got.drafted_tokens and (twist or config.greedy is False or got.kept_tokens == got.drafted_tokens)
        for r in (target, drafter):
            assert r.cache.free_pages() == [64] and not r.fed
            r.cache.check_consistency()


def test_an_end_token_stops_and_is_kept():
    want = generate(Runner(), Sampler(SamplerConfig(0.0), VOCAB), PROMPT, 60, sample=host_sample_row).generated_tokens
    for at in (0, 1, 2, 5, 11):
        seen = []
        got = run(Runner(), Runner(0.4), SamplerConfig(0.0), PROMPT, 4, 60, end=[want[at]], on_token=seen.append)
        first = want.index(want[at])
        assert got.generated_tokens == want[:first + 1] and got.stopped_by_end_token and seen == want[:first]


def test_drafts_behind_an_end_token_are_not_counted_as_kept():
    """An agreeing drafter, steps of five tokens of which the fifth is the target's own."""
    want = generate(Runner(), Sampler(SamplerConfig(0.0), VOCAB), PROMPT, 60, sample=host_sample_row).generated_tokens
    for at, kept in ((0, 1), (1, 2), (3, 4), (4, 4), (5, 5), (11, 10)):
        if want[at] in want[:at]:
            continue
        got = run(Runner(), Runner(), SamplerConfig(0.0), PROMPT, 4, 60, end=[want[at]])
        assert got.generated_tokens == want[:at + 1] and got.kept_tokens == kept and got.drafted_tokens == 4 * (at // 5 + 1)


def test_a_drafter_that_agrees_is_believed_at_any_temperature():
    """Equal distributions: every draft stays, so a step brings n_drafts + 1 tokens."""
    target = Runner()
    got = run(target, Runner(), SamplerConfig(1.3, seed=9), PROMPT, 4, 45)
    assert got.kept_tokens == got.drafted_tokens and len(got.generated_tokens) == 41
    assert sum(1 for entries in target.log if entries[0][2]) == 9              # 41 tokens, five a step


def test_the_first_tokens_frequencies_are_the_targets():
    """4,000 seeds: a frequency's standard deviation is at most 0.5 / 63; fifty of them within five (fixed numbers)."""
    target = Runner()
    target.open("x")
    row = target.step([SimpleNamespace(request="x", tokens=PROMPT, want=(len(PROMPT) - 1,))])[0].numpy()
    p = plain_drafts.softmax(row, 1.0)
    count = np.zeros(VOCAB)
    for seed in range(4000):
        tokens = run(Runner(), Runner(1.0), SamplerConfig(1.0, seed=seed), PROMPT, 1, len(PROMPT) + 1).generated_tokens
        count[tokens[0]] += 1
    assert abs(count / 4000 - p).max() < 5 * 0.5 / 4000 ** 0.5


def test_small_pools_and_contexts():
    want = generate(Runner(), Sampler(SamplerConfig(0.0), VOCAB), PROMPT, 40, sample=host_sample_row).generated_tokens
    got = run(Runner(n_pages=10), Runner(n_pages=3), SamplerConfig(0.0), PROMPT, 4, 40)        # the drafter's pages end at position 12, the target's with the request
    assert got.generated_tokens == want
    got = run(Runner(), Runner(max_positions=20), SamplerConfig(0.0), PROMPT, 4, 40)           # ... or its context
    assert got.generated_tokens == want
    got = run(Runner(max_rows=2), Runner(max_rows=2), SamplerConfig(0.0), PROMPT, 4, 40)       # steps of two rows: one draft each
    assert got.generated_tokens == want
    got = run(Runner(max_rows=1), Runner(), SamplerConfig(0.0), PROMPT, 4, 40)                 # no room for any
    assert got.generated_tokens == want and got.drafted_tokens == 0
    target, drafter = Runner(n_pages=3), Runner()
    with pytest.raises(OutOfPages):
        run(target, drafter, SamplerConfig(0.0), PROMPT, 4, 40)
    assert target.cache.free_pages() == [3] and drafter.cache.free_pages() == [64]


@pytest.mark.parametrize("config", [SamplerConfig(0.0), SamplerConfig(1.3, seed=9), SamplerConfig(0.9, top_k=6, seed=4)])
def test_what_was_proposed_before_the_drafters_pool_ran_out_is_judged(config):
    """12 positions: behind the prompt's 4 and the last token four proposals, then from position 9 three more; from position 12 on there is room for none."""
    target = Runner()
    got = run(target, Runner(n_pages=3), config, PROMPT, 4, 30)
    alone = run(Runner(), Runner(), config, PROMPT, 4, 30)
    proposed = [entries[0][1] - 1 for entries in target.log if entries[0][2]]
    assert len(got.generated_tokens) == 26 and got.drafted_tokens == sum(proposed) > 0 and proposed[0] == 4
    if config.greedy or config.top_k == 0:                    # an agreeing drafter: all stay
        assert proposed[:3] == [4, 3, 0] and got.kept_tokens == got.drafted_tokens == 7
    if config.greedy or config.top_k:
        assert got.generated_tokens == alone.generated_tokens


def test_refusals():
    target, sampler = Runner(), Sampler(SamplerConfig(0.0), VOCAB)
    with pytest.raises(ValueError, match="no tokens"):
        generate_with_drafts(target, Runner(), sampler, [])
    for n in (0, 65):
        with pytest.raises(ValueError, match="1 to 64"):
            generate_with_drafts(target, Runner(), sampler, PROMPT, n)
    with pytest.raises(ValueError, match="another runner"):
        generate_with_drafts(target, target, sampler, PROMPT)
    other = Runner()
    other.model = SimpleNamespace(spec=SimpleNamespace(vocab_size=VOCAB + 1))
    with pytest.raises(ValueError, match="same vocabulary"):
        generate_with_drafts(target, other, sampler, PROMPT)
    for one, two in ((Runner(windows=True), Runner()), (Runner(), Runner(windows=True))):
        with pytest.raises(ValueError, match="taken back"):
            generate_with_drafts(one, two, sampler, PROMPT)
    stateful = Runner()
    stateful.cache = CacheManager([PagedKvNeed(1, 2), StateNeed((3,))], [None, None], page_size=4, n_pages=64, max_requests=2, max_positions=96, allocate_storage=False)
    assert not stateful.cache.rewinds and target.cache.rewinds
    with pytest.raises(ValueError, match="taken back"):
        generate_with_drafts(stateful, Runner(), sampler, PROMPT)
    with pytest.raises(ValueError, match="does not fit"):
        generate_with_drafts(target, Runner(max_positions=4), sampler, PROMPT)


def test_models_on_two_devices_are_refused_before_anything_runs():
    target, drafter = Runner(), Runner()
    for r, device in ((target, "cuda:0"), (drafter, "cuda:1")):
        r.model = SimpleNamespace(spec=SimpleNamespace(vocab_size=VOCAB), device=torch.device(device))
    with pytest.raises(ValueError, match="lies on cuda:0 and the drafter on cuda:1"):
        generate_with_drafts(target, drafter, Sampler(SamplerConfig(0.0), VOCAB), PROMPT)
    assert not target.log and not drafter.log and not target.fed


def test_verify_rows_refuses():
    plain, drafts, logits = Sampler(SamplerConfig(1.0), VOCAB), torch.zeros((2, 3), dtype=torch.int32), torch.zeros(8, VOCAB)
    with pytest.raises(ValueError, match="samplers"):
        verify_rows_on_device(logits, drafts, [plain])
    with pytest.raises(ValueError, match="0 to 3"):
        verify_rows_on_device(logits, drafts, [plain] * 2, n_drafts=[1, 4])
    with pytest.raises(ValueError, match="rows of logits"):
        verify_rows_on_device(logits, drafts, [plain] * 2, n_drafts=[1, 3])
    with pytest.raises(ValueError, match="top-k or top-p"):
        verify_rows_on_device(logits, drafts, [plain, Sampler(SamplerConfig(1.0, top_k=4), VOCAB)])
