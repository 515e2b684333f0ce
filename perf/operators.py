"""Two operators of a server whose many requests share one model, as cases that can be timed:

  verify   drafted tokens are judged against the target's probabilities: each request brings some drafted tokens, the target's
           logits at their places and one place further, and the uniform numbers that decide.  Out come the tokens that stay, the one that is
           drawn behind them, and how many they are.
  adapt    low-rank adapters of many requests at once: every row of a batch gets scale * (x A^T) B^T of its own request's adapter on top of
           rows that are there.
  project  the same beside the projection that all rows share: x W^T + scale * (x A^T) B^T in one call.

Vocabularies and widths are those of `configs/` (128,256 and 32,000 tokens; 2,048 and 4,096 wide, 8,192 and 14,336 in the feed-forward) and
odd ones beside them.
"""
import math
import random

import numpy as np
import torch

own = False
DEVICE = "cuda:0"


def listed():
    return [
        # ---- verify
        # one user at a terminal with a small model drafting for a large one: latency
        dict(name="verify_b1", kind="verify", requests=1, drafts=4, vocab=128256, temperature=0.8, drafter="model", greedy=0, masked=0, ragged=False),
        # a few requests whose drafts come from a lookup in their own text (no probabilities), under a grammar that forbids most tokens
        dict(name="verify_b8_lookup", kind="verify", requests=8, drafts=3, vocab=128256, temperature=1.0, drafter="lookup", greedy=2, masked=2, ragged=True),
        # code completion: arg max throughout, a smaller vocabulary of an odd size
        dict(name="verify_b32_greedy", kind="verify", requests=32, drafts=5, vocab=32003, temperature=1.0, drafter="lookup", greedy=1, masked=0, ragged=False),
        # a full server: ragged numbers of drafts, some requests greedy
        dict(name="verify_b64", kind="verify", requests=64, drafts=7, vocab=128256, temperature=0.7, drafter="model", greedy=8, masked=4, ragged=True),
        # ---- adapt
        # one decoded token of one user
        dict(name="adapt_1", kind="adapt", rows="1", adapters=4, width=2048, slices="2048", rank=16, dtype="bfloat16", base="float32", result="float32"),
        # a decode step of a full server, every request with an adapter of its own, at the 8B feed-forward's way up
        dict(name="adapt_64_own", kind="adapt", rows="1x64", adapters=64, width=4096, slices="14336", rank=16, dtype="bfloat16", base="float32", result="float32"),
        # a portion of a prompt beside decoded rows, on the packed q/k/v projection
        dict(name="adapt_531_packed", kind="adapt", rows="1x19 301 211", adapters=21, width=4096, slices="4096 1024 1024", rank=24, dtype="bfloat16", base="float32",
             result="bfloat16"),
        # a step's whole budget of prompt rows of a few requests, at the 8B feed-forward's way down
        dict(name="adapt_4096", kind="adapt", rows="1777 64 1800 455", adapters=4, width=14336, slices="4096", rank=64, dtype="bfloat16", base="float32", result="float32"),
        # the 32-bit path, a rank of no round size
        dict(name="adapt_301_f32", kind="adapt", rows="1x3 298", adapters=3, width=2048, slices="2048", rank=10, dtype="float32", base="float32", result="float32"),
        # ---- project
        # a decode step with five drafted rows a request, at the 1B feed-forward's way down
        dict(name="project_40", kind="project", rows="5x8", adapters=8, width=8192, slices="2048", rank=16, dtype="bfloat16", base="float32", result="float32"),
        # a prompt through the 1B attention's way out, one adapter; rows stored as activations are
        dict(name="project_2048", kind="project", rows="2048", adapters=2, width=2048, slices="2048", rank=32, dtype="bfloat16", base="float32", result="bfloat16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.45:
        requests, vocab = _log_int(rng, 1, 64), _log_int(rng, 1000, 128256)
        return dict(kind="verify", requests=requests, drafts=rng.randint(1, 7), vocab=vocab, temperature=rng.choice([0.3, 0.7, 1.0, 1.3]),
                    drafter=rng.choice(["model", "model", "lookup"]), greedy=rng.choice([0, 0, 1, 3]), masked=rng.choice([0, 0, 3]), ragged=rng.random() < 0.5)
    kind = rng.choice(["adapt", "adapt", "project"])
    dtype = "bfloat16" if rng.random() < 0.8 else "float32"
    width = 8 * _log_int(rng, 32, 1024) if rng.random() < 0.8 else _log_int(rng, 256, 8192)
    parts = rng.choice([1, 1, 2, 3])
    slices = [_log_int(rng, 128, 8192 // parts) for _ in range(parts)]
    n = _log_int(rng, 1, 4096)
    rows = []
    while sum(rows) < n and len(rows) < 48:
        rows.append(min(n - sum(rows), 1 if rng.random() < 0.6 and n - sum(rows) < 1000 else _log_int(rng, 1, n)))
    if sum(rows) < n:
        rows.append(n - sum(rows))
    return dict(kind=kind, rows=" ".join(map(str, rows)), adapters=rng.randint(1, 24), width=width, slices=" ".join(map(str, slices)), rank=_log_int(rng, 4, 64) if rng.random() < 0.4 else rng.choice([8, 16, 32, 64]),
                dtype=dtype, base="float32", result=dtype if rng.random() < 0.5 else "float32")


# ------------------------------------------------------------------------------------------ inputs
def _numbers(text):
    """"1x3 298" -> [1, 1, 1, 298]."""
    out = []
    for word in text.split():
        value, _, times = word.partition("x")
        out += [int(value)] * int(times or 1)
    return out


def _generator(seed, n):
    return torch.Generator(device=DEVICE).manual_seed((seed * 1000003 + n) & 0x7fffffff)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _counts(case):
    """How many drafts each request brings: the case's own numbers, the same for every seed."""
    if not case["ragged"]:
        return [case["drafts"]] * case["requests"]
    rng = random.Random("%d %d %d" % (case["requests"], case["drafts"], case["vocab"]))
    return [case["drafts"] if i == 0 else rng.randint(0, case["drafts"]) for i in range(case["requests"])]


def _prepare_verify(case, seed):
    R, K, V, g = case["requests"], case["drafts"], case["vocab"], _generator(seed, 1)
    counts = _counts(case)
    n_rows = sum(counts) + R
    first = np.cumsum([0] + [n + 1 for n in counts[:-1]])
    temperature = torch.full((R,), case["temperature"], device=DEVICE)
    if case["greedy"]:                                                  # every so manieth request takes the arg max
        temperature[::case["greedy"]] = 0.0
    # logits as language models make them: a wide body and a few tokens far above it, and a drafter that mostly agrees
    logits = 2.0 * _randn(g, n_rows, V)
    heads = torch.randint(0, V, (n_rows, 8), generator=g, device=DEVICE)
    logits.scatter_add_(1, heads, 6.0 + 2.5 * _randn(g, n_rows, 8))
    if case["masked"]:                                                  # a grammar: most tokens of some requests are forbidden
        allowed = torch.rand(n_rows, V, generator=g, device=DEVICE) < 0.02
        allowed[:, 0] = True
        owner = torch.repeat_interleave(torch.arange(R, device=DEVICE), torch.tensor([n + 1 for n in counts], device=DEVICE))
        logits.masked_fill_((owner % case["masked"] == 0)[:, None] & ~allowed, -math.inf)
    rows = torch.tensor([[int(first[r]) + min(j, counts[r]) for j in range(K)] for r in range(R)], device=DEVICE)
    draft_logits = None
    t = torch.where(temperature > 0, temperature, 1.0)[:, None, None]
    if case["drafter"] == "model":
        draft_logits = logits[rows] + 0.8 * _randn(g, R, K, V)
        noise = torch.rand(R, K, V, generator=g, device=DEVICE).clamp_min_(1e-9).log_().neg_().log_().neg_()
        drafts = (draft_logits / t + noise).argmax(-1)                  # drawn from the drafter's own softmax
    else:                                                               # a lookup: often what the target finds likely
        likely = (logits[rows] + 0.8 * _randn(g, R, K, V)).argmax(-1)
        drafts = torch.where(torch.rand(R, K, generator=g, device=DEVICE) < 0.8, likely, torch.randint(0, V, (R, K), generator=g, device=DEVICE))
    uniform = torch.rand(R, K + 1, generator=g, device=DEVICE)
    return dict(case=case, logits=logits, draft_logits=draft_logits, drafts=drafts.int().contiguous(), temperature=temperature, uniform=uniform,
                n_drafts=torch.tensor(counts, dtype=torch.int32, device=DEVICE), first_row=torch.tensor(first, dtype=torch.int32, device=DEVICE),
                tokens=torch.empty((R, K + 1), dtype=torch.int32, device=DEVICE), counts=torch.empty(R, dtype=torch.int32, device=DEVICE))


def _prepare_adapt(case, seed):
    rows, slices, K, r, E = _numbers(case["rows"]), _numbers(case["slices"]), case["width"], case["rank"], case["adapters"]
    n, O, S = sum(rows), sum(slices), len(slices)
    dtype, result, g = getattr(torch, case["dtype"]), getattr(torch, case["result"]), _generator(seed, 2)
    # requests take adapters in no order; where there are enough rows some request has none
    rng = random.Random(seed)
    names = [rng.randrange(E) for _ in rows] if E < len(rows) else rng.sample(range(E), len(rows))
    if len(names) > 4:
        names[len(names) // 2] = -1
    per_row = np.repeat(np.asarray(names, dtype=np.int32), rows)
    state = dict(case=case, x=_randn(g, n, K).to(dtype), a=(_randn(g, E, S * r, K) / K ** 0.5).to(dtype), b=(0.3 / r ** 0.5 * _randn(g, E, O, r)).to(dtype),
                 scales=torch.rand(E, generator=g, device=DEVICE) + 0.5, ids=torch.from_numpy(per_row).to(DEVICE),
                 rows_of=[(e, torch.from_numpy(np.flatnonzero(per_row == e)).to(DEVICE)) for e in range(E) if (per_row == e).any()],
                 slices=None if S == 1 else tuple(slices), out=torch.empty((n, O), dtype=result, device=DEVICE))
    if case["kind"] == "project":
        state["weight"] = (_randn(g, O, K) / K ** 0.5).to(dtype)
    else:
        state["base"] = _randn(g, n, O).to(getattr(torch, case["base"]))
    return state


def prepare(case, seed):
    return _prepare_verify(case, seed) if case["kind"] == "verify" else _prepare_adapt(case, seed)


# -------------------------------------------------------------------------------------------- run
def _plain_verify(s):
    """u_j q_j(x_j) < p_j(x_j) keeps draft x_j; the first that falls is replaced by a draw from max(p - q, 0), behind the last that stays comes a
    draw from p.  Probabilities and running sums in 64 bits: a draw compares against sums over the whole vocabulary."""
    logits, drafts, uniform = s["logits"], s["drafts"].long(), s["uniform"].double()
    R, K = drafts.shape
    V, dev = logits.shape[1], logits.device
    counts, greedy = s["n_drafts"].long(), ~(s["temperature"] > 0)
    place = torch.arange(K + 1, device=dev)
    rows = s["first_row"].long()[:, None] + torch.minimum(place[None, :], counts[:, None])
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None, None]

    def softmax(l):
        e = torch.exp((l.double() - l.amax(-1, keepdim=True).double()) / t)
        return e / e.sum(-1, keepdim=True)

    target = logits[rows]                                                       # [R, K + 1, V]
    top = torch.where(target == target.amax(-1, keepdim=True), torch.arange(V, device=dev), V).amin(-1)
    p = softmax(target)
    del target
    p_x = p[:, :K].gather(2, drafts[:, :, None])[:, :, 0]
    q = None
    if s["draft_logits"] is not None:
        q = softmax(s["draft_logits"])
        q_x = q.gather(2, drafts[:, :, None])[:, :, 0]
    else:
        q_x = torch.ones_like(p_x)
    stays = torch.where(greedy[:, None], drafts == top[:, :K], uniform[:, :K] * q_x < p_x) & (place[None, :K] < counts[:, None])
    kept = stays.long().cumprod(1).sum(1)                                       # [R]
    one = torch.arange(R, device=dev)
    last, fell = p[one, kept], kept < counts
    at = kept.clamp_max(K - 1)
    if q is not None:
        rest = (last - torch.where(fell[:, None], q[one, at], 0.0)).clamp_min(0.0)
    else:
        rest = last.clone()
        rest[one, drafts[one, at]] = torch.where(fell, 0.0, rest[one, drafts[one, at]])
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, last)
    sums = rest.cumsum(-1)
    index = torch.arange(V, device=dev)
    hit = torch.where(sums > uniform[:, K, None] * sums[:, -1:], index, V).amin(-1)
    drawn = torch.where(hit < V, hit, torch.where(rest > 0, index, 0).amax(-1))
    drawn = torch.where(greedy, top[one, kept], drawn)
    tokens = torch.where(place[None, :] < kept[:, None], torch.cat([drafts, drafts[:, :1]], 1), torch.where(place[None, :] == kept[:, None], drawn[:, None], -1))
    return tokens.int(), (kept + 1).int()


def _plain_adapt(s):
    x, r, result = s["x"].float(), s["b"].shape[2], s["out"].dtype
    O = s["b"].shape[1]
    out = x @ s["weight"].float().t() if "weight" in s else s["base"].float()
    slices = s["slices"] or (O,)
    edges = np.cumsum((0,) + tuple(slices))
    if "weight" not in s:
        out = out.clone()
    for e, rows in s["rows_of"]:
        t = s["scales"][e] * (x[rows] @ s["a"][e].float().t())
        b = s["b"][e].float()
        out[rows] += torch.cat([t[:, i * r:(i + 1) * r] @ b[edges[i]:edges[i + 1]].t() for i in range(len(slices))], 1)
    return out.to(result)


def run(state):
    if not own:
        return _plain_verify(state) if state["case"]["kind"] == "verify" else _plain_adapt(state)
    if state["case"]["kind"] == "verify":
        from geneinfer_amd.kernels import ops
        return ops.verify_drafts(state["logits"], state["drafts"], state["temperature"], state["uniform"], state["tokens"], state["counts"],
                                 draft_logits=state["draft_logits"], n_drafts=state["n_drafts"], first_row=state["first_row"])
    if state["case"]["kind"] == "adapt":
        from geneinfer_amd.kernels import ops
        return ops.adapters_add(state["x"], state["a"], state["b"], state["ids"], state["out"], scales=state["scales"], base=state["base"], slices=state["slices"])
    from geneinfer_amd.parts.linear import RowAdapters, linear
    return linear(state["x"], state["weight"], state["out"], adapters=RowAdapters(state["a"], state["b"], state["ids"], state["scales"], state["slices"]))


# ------------------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "verify":
        counts, V = _counts(case), case["vocab"]
        read = sum(n + 1 for n in counts)
        if case["drafter"] == "model":                                  # (an arg max asks for none of the drafter's)
            read += sum(n for i, n in enumerate(counts) if not case["greedy"] or i % case["greedy"])
        return dict(bytes=4 * read * V, flops=4 * read * V)
    rows, slices, K, r = _numbers(case["rows"]), _numbers(case["slices"]), case["width"], case["rank"]
    n, O, S = sum(rows), sum(slices), len(slices)
    size = {"bfloat16": 2, "float32": 4}
    some = min(case["adapters"], len(rows))                     # adapters that rows ask for
    moved = n * K * size[case["dtype"]] + some * r * (S * K + O) * size[case["dtype"]] + n * O * size[case["result"]]
    flops = 2 * n * r * (S * K + O)
    if case["kind"] == "project":
        return dict(bytes=moved + O * K * size[case["dtype"]], flops=flops + 2 * n * K * O)
    return dict(bytes=moved + n * O * size[case["base"]], flops=flops)


# ------------------------------------------------------------------------------------------ exact
def _exact_verify(s):
    """Request by request and token by token, in numpy's 64 bits."""
    logits, drafts, uniform = s["logits"].cpu().numpy(), s["drafts"].cpu().numpy(), s["uniform"].cpu().numpy().astype(np.float64)
    first, counts, temps = s["first_row"].tolist(), s["n_drafts"].tolist(), s["temperature"].cpu().numpy().astype(np.float64)
    K = drafts.shape[1]
    tokens, lengths = np.full((len(counts), K + 1), -1, dtype=np.int32), np.zeros(len(counts), dtype=np.int32)

    def distribution(row, t):
        w = np.exp((row.astype(np.float64) - float(row.max())) / t)
        return w / w.sum()

    for r, n in enumerate(counts):
        j = 0
        while True:
            row = logits[first[r] + j]
            if not temps[r] > 0:
                best = int(np.argmax(row))
                if j < n and drafts[r, j] == best:
                    tokens[r, j], j = best, j + 1
                    continue
                tokens[r, j] = best
                break
            p = distribution(row, temps[r])
            left = p
            if j < n:
                x = int(drafts[r, j])
                if s["draft_logits"] is None:
                    q = np.zeros_like(p)
                    q[x] = 1.0
                else:
                    q = distribution(s["draft_logits"][r, j].cpu().numpy(), temps[r])
                if uniform[r, j] * q[x] < p[x]:
                    tokens[r, j], j = x, j + 1
                    continue
                left = np.maximum(p - q, 0.0)
                if not left.sum() > 0:
                    left = p
            running = np.cumsum(left)
            i = int(np.searchsorted(running, uniform[r, K] * running[-1], side="right"))
            tokens[r, j] = i if i < len(running) else int(np.flatnonzero(left)[-1])
            break
        lengths[r] = j + 1
    return torch.from_numpy(tokens), torch.from_numpy(lengths)


def _exact_adapt(s):
    """x (W + scale B A)^T with the adapter's whole matrix made first, in 64 bits."""
    x, ids = s["x"].double(), s["ids"]
    E, O, r = s["b"].shape
    y = s["base"].double() if "base" in s else x @ s["weight"].double().t()
    slices, result = s["slices"] or (O,), torch.empty_like(y)
    for e in range(-1, E):
        mine = (ids == e).nonzero()[:, 0]
        if not len(mine):
            continue
        result[mine] = y[mine]
        start = 0
        for i, columns in enumerate(slices if e >= 0 else ()):
            whole = s["scales"][e].double() * (s["b"][e, start:start + columns].double() @ s["a"][e, i * r:(i + 1) * r].double())
            result[mine, start:start + columns] += x[mine] @ whole.t()
            start += columns
    return result


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_verify(state) if case["kind"] == "verify" else _exact_adapt(state)
