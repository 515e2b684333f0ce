"""Generation with a drafter on the device: models of the tiny Llama shapes, drafts judged by the kernels."""
import numpy as np
import pytest
import torch

import plain_drafts
from model_folders import CONFIGS, PAGE_SIZE, write_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for name, seed in (("target", 41), ("drafter", 42)):
        out[name] = tmp_path_factory.mktemp(name)
        write_model(out[name], CONFIGS["B"], seed=seed)
    return out


def llm(folder, dtype="float32", **kw):
    import geneinfer_amd as gi
    return gi.LLM(folder, dtype=dtype, page_size=PAGE_SIZE["B"], max_tokens=256, max_running=2, **kw)


def prompt(n, seed=3):
    return np.random.default_rng(seed).integers(0, CONFIGS["B"]["vocab_size"], n).tolist()


@pytest.mark.parametrize("settings", [dict(temperature=0.0), dict(temperature=0.9, top_k=7), dict(temperature=1.1, top_p=0.7, top_k=20)])
def test_tokens_are_those_without_a_drafter(folders, settings):
    """The 32-bit path: a row's logits have the same bits in a step of several rows."""
    target, drafter = llm(folders["target"]), llm(folders["drafter"])
    for n, n_drafts in ((1, 3), (9, 1), (14, 6)):
        p = prompt(n)
        want = target.generate(p, steps=n + 30, seed=7, **settings)
        got = target.generate(p, steps=n + 30, seed=7, drafter=drafter, n_drafts=n_drafts, **settings)
        assert got.generated_tokens == want.generated_tokens and got.drafted_tokens > 0
        assert target.runner.cache.free_pages() == drafter.runner.cache.free_pages()
        assert target.generate(p, steps=n + 12, seed=8, **settings).generated_tokens == target.generate(p, steps=n + 12, seed=8, drafter=drafter, **settings).generated_tokens


@pytest.mark.parametrize("temperature", [0.0, 0.8, 1.5])
def test_the_same_model_as_drafter_is_always_right(folders, temperature):
    target, drafter = llm(folders["target"]), llm(folders["target"])
    got = target.generate(prompt(8), steps=47, temperature=temperature, drafter=drafter, n_drafts=4)
    assert got.kept_tokens == got.drafted_tokens == 32 and len(got.generated_tokens) == 40 and got.decode_steps == 7


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_drafts_are_judged_by_the_logits_of_the_steps(folders, dtype, monkeypatch):
    """Every judgement of a request against the plain one from the same logits, proposals and numbers."""
    import sys
    module = sys.modules["geneinfer_amd.engine.generate"]
    target, drafter = llm(folders["target"], dtype), llm(folders["drafter"], dtype)
    judged = []
    original = module.verify_rows

    def watched(logits, drafts, samplers, draft_logits=None, n_drafts=None):
        state = samplers[0].stream.state
        got = original(logits, drafts, samplers, draft_logits, n_drafts)
        after, samplers[0].stream.state = samplers[0].stream.state, state
        k = drafts.shape[1]
        uniform = np.array([[samplers[0].next_uniform() for _ in range(k + 1)]], dtype=np.float32)
        assert samplers[0].stream.state == after
        tokens, counts = plain_drafts.verify(logits.cpu().numpy(), drafts.cpu().numpy(), [samplers[0].temperature], uniform, None if draft_logits is None else draft_logits.cpu().numpy())
        assert got == [tokens[0, :counts[0]].tolist()]
        judged.append(counts[0])
        return got
    monkeypatch.setattr(module, "verify_rows", watched)
    got = target.generate(prompt(11), steps=60, temperature=0.9, seed=5, drafter=drafter, n_drafts=5)
    assert len(got.generated_tokens) == 50 == sum(judged) and got.kept_tokens == sum(judged) - len(judged)
    assert 0 < got.kept_tokens < got.drafted_tokens


def test_verify_rows_of_many_requests(folders):
    from geneinfer_amd.sampling import Sampler, SamplerConfig, verify_rows
    vocab, counts = 601, [3, 0, 2, 3, 1]
    g = torch.Generator().manual_seed(2)
    logits = (2 * torch.randn(sum(counts) + 5, vocab, generator=g)).to("cuda:0")
    drafts = torch.randint(0, vocab, (5, 3), generator=g).int()
    first = np.cumsum([0] + [c + 1 for c in counts[:-1]]).astype(np.int32)
    for r, c in enumerate(counts):
        for j in range(c):
            if (r + j) % 3:
                drafts[r, j] = int(logits[first[r] + j].argmax())
    make = lambda: [Sampler(SamplerConfig(t, seed=i), vocab) for i, t in enumerate((0.7, 0.9, 0.0, 1.2, 0.3))]
    uniform = np.zeros((5, 4), np.float32)
    for r, s in enumerate(make()):
        if not s.config.greedy:
            uniform[r, list(range(counts[r])) + [3]] = [s.next_uniform() for _ in range(counts[r] + 1)]
    tokens, n = plain_drafts.verify(logits.cpu().numpy(), drafts.numpy(), [0.7, 0.9, 0.0, 1.2, 0.3], uniform, None, counts, first)
    assert verify_rows(logits, drafts.to("cuda:0"), make(), n_drafts=counts) == [row[:c].tolist() for row, c in zip(tokens, n)]


def test_the_numbers_of_many_requests_do_not_wait_for_the_device():
    """600 requests bring 6,600 numbers.  The device has some hundreds of milliseconds of products before it; the call returns while they run, whichever buffers it takes."""
    from geneinfer_amd.sampling import Sampler, SamplerConfig, verify_rows_on_device
    n, k, vocab = 600, 7, 64
    logits, drafts = torch.randn(n * (k + 1), vocab, device="cuda:0"), torch.zeros((n, k), dtype=torch.int32, device="cuda:0")
    samplers = [[Sampler(SamplerConfig(1.0, seed=i), vocab) for i in range(n)] for _ in range(3)]
    want = verify_rows_on_device(logits, drafts, samplers[0])                     # (the library and its memory are there from now on)
    a = torch.randn(8192, 8192, device="cuda:0", dtype=torch.bfloat16)
    b = a @ a
    torch.cuda.synchronize()
    for _ in range(400):
        torch.mm(a, a, out=b)
    busy = torch.cuda.Event()
    busy.record()
    got = [verify_rows_on_device(logits, drafts, s) for s in samplers[1:]]
    assert not busy.query()
    for tokens, counts in got:
        assert torch.equal(tokens, want[0]) and torch.equal(counts, want[1])


def test_a_model_with_memories_is_refused(folders):
    import geneinfer_amd as gi
    target = llm(folders["target"])
    from geneinfer_amd.config import parse_config
    import json
    from pathlib import Path
    config = parse_config(json.loads((Path(__file__).resolve().parent.parent / "configs" / "fekorax-small.json").read_text()))
    recurrent = gi.LLM(gi.random_model(config, 0), max_tokens=64, max_running=2)
    with pytest.raises(ValueError):
        target.generate(prompt(4), steps=9, drafter=recurrent)


def test_real_models_with_memories_are_refused_on_either_side(folders):
    """Of one vocabulary, so that the memories are what is refused."""
    import json
    from pathlib import Path
    import geneinfer_amd as gi
    from geneinfer_amd.config import parse_config
    target = llm(folders["target"])
    config = json.loads((Path(__file__).resolve().parent.parent / "configs" / "fekorax-small.json").read_text())
    config["vocab"] = target.model.spec.vocab_size
    recurrent = gi.LLM(gi.random_model(parse_config(config), 0), max_tokens=64, max_running=2)
    with pytest.raises(ValueError, match="the drafter keeps a state or gives pages back; .* taken back"):
        target.generate(prompt(4), steps=9, drafter=recurrent)
    with pytest.raises(ValueError, match="the target keeps a state or gives pages back; .* taken back"):
        recurrent.generate(prompt(4), steps=9, drafter=target)
