"""Drafted tokens judged on the device against the same in numpy's 64 bits, token for token."""
import numpy as np
import pytest
import torch

import plain_drafts

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
GUARD = -123


def ops():
    from geneinfer_amd.kernels import ops as o
    return o


def case(n, k, vocab, *, temperature=0.8, drafter=True, seed=0, ragged=False, scale=2.0, noise=0.7):
    """Drafts as a drafter that mostly agrees makes them."""
    rng = np.random.default_rng(seed + 7919 * n + 104729 * k + vocab)
    n_drafts = rng.integers(0, k + 1, n).astype(np.int32) if ragged else np.full(n, k, dtype=np.int32)
    first = np.concatenate([[0], np.cumsum(n_drafts + 1)[:-1]]).astype(np.int32)
    logits = (scale * rng.standard_normal((int(n_drafts.sum()) + n, vocab))).astype(np.float32)
    logits[np.arange(len(logits)), rng.integers(0, vocab, len(logits))] += np.float32(8.0)
    t = np.full(n, temperature, dtype=np.float32)
    draft_logits = np.zeros((n, k, vocab), dtype=np.float32)
    drafts = np.zeros((n, k), dtype=np.int32)
    for r in range(n):
        for j in range(k):
            draft_logits[r, j] = logits[first[r] + min(j, n_drafts[r])] + noise * rng.standard_normal(vocab)
            drafts[r, j] = plain_drafts.draw(plain_drafts.softmax(draft_logits[r, j], temperature if temperature > 0 else 1.0), rng.random())
    uniform = rng.random((n, k + 1)).astype(np.float32)
    return dict(logits=logits, drafts=drafts, temperature=t, uniform=uniform, draft_logits=draft_logits if drafter else None, n_drafts=n_drafts, first_row=first)


def on_device(values):
    return None if values is None else torch.from_numpy(np.ascontiguousarray(values)).to(DEV)


def run(c, **over):
    n, k = c["drafts"].shape
    room = torch.full((n + 2, k + 1), GUARD, dtype=torch.int32, device=DEV)
    counts = torch.full((n + 2,), GUARD, dtype=torch.int32, device=DEV)
    given = {name: on_device(values) for name, values in c.items()}
    given.update(over)
    got = ops().verify_drafts(given["logits"], given["drafts"], given["temperature"], given["uniform"], room[1:-1], counts[1:-1], draft_logits=given["draft_logits"],
                              n_drafts=given["n_drafts"], first_row=given["first_row"])
    assert got[0].data_ptr() == room[1:-1].data_ptr()
    assert (room[0] == GUARD).all() and (room[-1] == GUARD).all() and counts[0] == counts[-1] == GUARD
    return room[1:-1].cpu().numpy(), counts[1:-1].cpu().numpy()


def check(c, **over):
    got, want = run(c, **over), plain_drafts.verify(**c)
    assert np.array_equal(got[1], want[1]), (got, want)
    assert np.array_equal(got[0], want[0]), (got, want)
    return got


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("n,k,vocab", [(1, 1, 1), (1, 4, 2), (3, 2, 7), (2, 3, 63), (5, 4, 256), (4, 3, 1001), (2, 5, 4095), (2, 5, 4096), (2, 5, 4097), (3, 2, 8192), (2, 7, 32003),
                                       (1, 4, 128256), (1, 2, 300007), (40, 1, 513)])
def test_against_64_bits(n, k, vocab, drafter):
    for seed in range(3):
        check(case(n, k, vocab, drafter=drafter, seed=seed))


@pytest.mark.parametrize("temperature", [0.05, 0.3, 1.0, 4.0, 1e-30, float("inf")])
def test_temperatures(temperature):
    c = case(4, 3, 1500, seed=5)
    c["temperature"][:] = temperature
    check(c)


@pytest.mark.parametrize("drafter", [True, False])
def test_ragged_numbers_of_drafts_and_greedy_rows_among_others(drafter):
    for seed in range(4):
        c = case(17, 6, 2100, drafter=drafter, ragged=True, seed=seed)
        c["temperature"][::3] = 0.0
        c["temperature"][1] = -1.0
        c["temperature"][4] = float("nan")                    # (neither is greater than 0: the arg max)
        for r in range(0, 17, 3):                             # what an arg max would draft, for some places
            for j in range(0, int(c["n_drafts"][r]), 2):
                c["drafts"][r, j] = int(np.argmax(c["logits"][c["first_row"][r] + j]))
        check(c)


def test_every_draft_may_stay_and_none():
    c = case(6, 4, 3000, noise=0.0, seed=2)
    c["uniform"][:, :4] = np.float32(1 - 2 ** -24)            # drafts drawn from the target's own distribution stay whatever the number
    assert (check(c)[1] == 5).all()
    c = case(6, 4, 3000, drafter=False, seed=3)
    c["drafts"][:, 0] = 17
    c["logits"][c["first_row"], 17] = -np.inf                 # impossible tokens
    assert (check(c)[1] == 1).all()


def test_no_drafts_is_a_draw():
    c = case(5, 0, 5000, seed=4)
    c["draft_logits"] = None
    got = check(c)
    from geneinfer_amd.kernels import ops as o
    drawn = torch.empty(5, dtype=torch.int32, device=DEV)
    o.sample_temperature(on_device(c["logits"]), on_device(c["temperature"]), on_device(c["uniform"][:, 0].copy()), drawn)
    assert (drawn.cpu().numpy() == got[0][:, 0]).all()        # (numbers far from every boundary: 32-bit weights draw the same)


def test_equal_logits_ties_and_the_ends_of_the_unit_interval():
    c = case(6, 2, 4099, drafter=False, seed=6)
    c["logits"][:] = 1.25
    c["uniform"][:, 2] = [0.0, 1 - 2 ** -24, 0.5, 1.0, 0.25, 0.0]
    check(c)
    c["temperature"][:] = 0.0                                 # the lowest index of equal ones
    assert (check(c)[0][:, 0] == 0).all()


def test_a_goal_between_two_roundings_of_one_sum_draws_no_masked_token():
    """With a, b, c the weights e^l of the first three tokens that have any, (b + c) + a rounds to the uniform number given and c + (a + b) to the next 64-bit number: the goal lies at
    the end of the third's share by one order of additions and just below it by another, with a run of masked tokens behind.  The third or the fourth may be drawn, nothing else."""
    vocab = 300007                                            # 74 runs of 4,096, two a lane of the draw
    weighs = [5, 2 * 4096, 4 * 4096 + 77, 9 * 4096 + 9, vocab - 1]
    logits = np.full((1, vocab), -np.inf, dtype=np.float32)
    logits[0, weighs] = [-40.48126220703125, -40.11710739135742, -40.94380187988281, -40.5, 0.0]
    tokens, counts = run(dict(logits=logits, drafts=np.zeros((1, 0), np.int32), temperature=np.ones(1, np.float32), uniform=np.array([[8.057590335116807e-18]], np.float32),
                              draft_logits=None, n_drafts=None, first_row=None))
    assert counts[0] == 1 and tokens[0, 0] in weighs[2:4]


def test_masked_rows_infinities_and_nan():
    c = case(9, 3, 4200, seed=7)
    first = c["first_row"]
    c["logits"][first[0]:first[0] + 4, :4100] = -np.inf       # a whole run of the row and more is masked
    c["draft_logits"][0, :, 50:] = -np.inf                    # the drafter allows what the target forbids
    c["drafts"][0] = 7
    c["logits"][first[1]:first[1] + 4] = -np.inf              # nothing left
    c["logits"][first[2], 4199] = np.inf
    c["logits"][first[3], [5, 4100]] = np.inf                 # two that share all mass
    c["logits"][first[4], ::2] = np.nan
    c["logits"][first[5]:first[5] + 4] = np.nan
    c["draft_logits"][6] = -np.inf                            # a drafter without a distribution: its draft stays where p has it
    c["draft_logits"][7, :, 11] = np.inf
    c["logits"][first[8], :] = np.finfo(np.float32).min       # a mask of the type's lowest value everywhere but at one token
    c["logits"][first[8], 4150] = 3.0
    check(c)
    c["temperature"][:] = 0.0
    check(c)
    c["temperature"][:] = float("inf")
    check(c)
    c["draft_logits"], c["temperature"] = None, np.full(9, 0.7, dtype=np.float32)
    check(c)


def test_rows_without_a_token():
    """At a temperature no draft stays and the token is 0; the arg max of such a row is 0, as without drafts, so a draft of 0 stays and the next row is asked."""
    from geneinfer_amd.kernels import ops as o
    c = case(2, 2, 500, drafter=False, seed=15)
    c["logits"][[0, 1]], c["logits"][3] = -np.inf, np.nan
    c["logits"][[2, 4], 77], c["drafts"][:] = 40.0, [[0, 0], [5, 0]]
    assert check(c)[0].tolist() == [[0, -1, -1], [0, -1, -1]]
    c["temperature"][:] = 0.0
    assert check(c)[0].tolist() == [[0, 0, 77], [0, -1, -1]]
    alone = torch.empty(6, dtype=torch.int32, device=DEV)
    assert o.argmax(on_device(np.where(np.isnan(c["logits"]), -np.inf, c["logits"]).astype(np.float32)), alone)[:5].tolist() == [0, 0, 77, 0, 77]


@pytest.mark.parametrize("drafter", [True, False])
def test_drafts_outside_the_vocabulary_fall(drafter):
    c = case(4, 3, 777, drafter=drafter, seed=8, noise=0.0)
    c["drafts"][0, 0], c["drafts"][1, 1], c["drafts"][2, 0], c["drafts"][3, 2] = -1, 777, 2 ** 31 - 1, -2 ** 31
    check(c)
    c["temperature"][:] = 0.0
    check(c)


def test_requests_whose_rows_are_not_there_get_nothing():
    c = case(5, 2, 300, seed=9)
    c["first_row"] = np.array([0, 13, -1, 2 ** 31 - 1, 12], dtype=np.int32)       # 15 rows: the second has its three, the last two of the list run out
    got = check(c)
    assert got[1][2] == got[1][3] == 0 and (got[0][2] == -1).all()
    c["first_row"][:] = [12, 12, 13, 14, 0]
    check(c)
    c["n_drafts"] = np.array([-5, 99, 0, 0, 2], dtype=np.int32)                   # held to 0 .. K
    check(c)


def test_nothing_left_beside_the_drafter_falls_back_on_p():
    c = case(2, 1, 100, seed=10, noise=0.0)
    c["drafts"][:, 0] = [-1, 100]                             # fall as no tokens; p - q is 0 everywhere
    check(c)


def test_strides():
    c = case(3, 2, 1001, seed=11)
    wide = torch.full((9, 1009), 50.0, device=DEV)
    wide[:, :1001] = on_device(c["logits"])
    deep = torch.full((3, 4, 1100), 50.0, device=DEV)
    deep[:, 1:3, 5:1006] = on_device(c["draft_logits"])
    check(c, logits=wide[:, :1001], draft_logits=deep[:, 1:3, 5:1006])
    shared = case(3, 2, 64, seed=12)
    shared["draft_logits"][:] = shared["draft_logits"][:1, :1]                    # one drafter's row for all, broadcast
    check(shared, draft_logits=on_device(shared["draft_logits"][0, 0]).expand(3, 2, 64))


def test_defaults_are_k_drafts_each_in_order():
    c = case(3, 4, 900, seed=13)
    want = run(c)
    c["n_drafts"] = c["first_row"] = None
    got = check(c)
    assert np.array_equal(want[0], got[0])


def test_no_requests():
    o = ops()
    e = torch.empty
    tokens, counts = e((0, 3), dtype=torch.int32, device=DEV), e(0, dtype=torch.int32, device=DEV)
    o.verify_drafts(e((0, 9), device=DEV), e((0, 2), dtype=torch.int32, device=DEV), e(0, device=DEV), e((0, 3), device=DEV), tokens, counts)


def test_tokens_are_distributed_as_the_target_has_them():
    """The first token's frequencies over many numbers, whoever drafts: 40,000 requests of a vocabulary of 6; a frequency's standard deviation
    is at most 0.5 / 200 = 0.0025, and 24 of them stay within five of those but for one run in some 70,000 (these numbers are fixed)."""
    n, vocab = 40000, 6
    rng = np.random.default_rng(21)
    p_l, q_l = rng.standard_normal(vocab).astype(np.float32), rng.standard_normal(vocab).astype(np.float32)
    p = plain_drafts.softmax(p_l, 0.9)
    for drafter in (True, False):
        q = plain_drafts.softmax(q_l, 0.9)
        drafts = rng.choice(vocab, size=(n, 1), p=q).astype(np.int32)
        c = dict(logits=np.broadcast_to(p_l, (2 * n, vocab)).copy(), drafts=drafts, temperature=np.full(n, 0.9, np.float32), uniform=rng.random((n, 2)).astype(np.float32),
                 draft_logits=np.broadcast_to(q_l, (n, 1, vocab)).copy() if drafter else None, n_drafts=None, first_row=None)
        tokens, counts = run(c)
        assert abs(np.bincount(tokens[:, 0], minlength=vocab) / n - p).max() < 5 * 0.0025
        second = tokens[counts == 2, 1]
        assert abs(np.bincount(second, minlength=vocab) / len(second) - p).max() < 5 * 0.5 / len(second) ** 0.5


def test_captured_and_replayed_with_other_inputs():
    o = ops()
    cs = [case(6, 4, 5003, seed=s, ragged=False) for s in range(3)]
    held = {name: on_device(v) for name, v in cs[0].items()}
    tokens, counts = torch.empty((6, 5), dtype=torch.int32, device=DEV), torch.empty(6, dtype=torch.int32, device=DEV)

    def call():
        o.verify_drafts(held["logits"], held["drafts"], held["temperature"], held["uniform"], tokens, counts, draft_logits=held["draft_logits"], n_drafts=held["n_drafts"],
                        first_row=held["first_row"])

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for c in (*cs, *cs):
        for name, v in c.items():
            held[name].copy_(on_device(v))
        graph.replay()
        got = tokens.cpu().numpy().copy(), counts.cpu().numpy().copy()
        want = plain_drafts.verify(**c)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        call()                                                # the program's own work between the replays
        assert np.array_equal(tokens.cpu().numpy(), want[0])


def test_two_streams_at_once():
    cs = [case(8, 3, 20011, seed=s) for s in range(2)]
    given = [{name: on_device(v) for name, v in c.items()} for c in cs]
    outs = [(torch.empty((8, 4), dtype=torch.int32, device=DEV), torch.empty(8, dtype=torch.int32, device=DEV)) for _ in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, (tokens, counts), s in zip(given, outs, streams):
            with torch.cuda.stream(s):
                ops().verify_drafts(g["logits"], g["drafts"], g["temperature"], g["uniform"], tokens, counts, draft_logits=g["draft_logits"], n_drafts=g["n_drafts"], first_row=g["first_row"])
    torch.cuda.synchronize()
    for c, (tokens, counts) in zip(cs, outs):
        want = plain_drafts.verify(**c)
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(counts.cpu().numpy(), want[1])


def test_offsets_beyond_32_bits():
    """The last request's rows begin 2^31 numbers and more behind the first's, and so do the drafter's."""
    vocab, k, n = 128256, 1, 3
    c = case(n, k, vocab, seed=14)
    rows = 2 ** 31 // vocab + 20
    logits = torch.zeros((rows, vocab), device=DEV)
    first = np.array([0, rows // 2, rows - 2], dtype=np.int32)
    for r in range(n):
        logits[int(first[r]):int(first[r]) + 2] = on_device(c["logits"][2 * r:2 * r + 2])
    big = torch.empty_strided((n, k, vocab), (rows * vocab, vocab, 1), device=DEV)
    big.copy_(on_device(c["draft_logits"]))
    want = plain_drafts.verify(**c)
    given = dict(c, first_row=first)
    got = run(given, logits=logits, draft_logits=big)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_the_most_requests_and_tokens_and_one_more():
    n = 65535
    c = case(3, 1, 5)
    many = {name: None if values is None else np.concatenate([values] * (n // 3)) for name, values in c.items()}
    many["first_row"] = (c["first_row"][None] + 6 * np.arange(n // 3, dtype=np.int32)[:, None]).reshape(-1)
    got, few = run(many), plain_drafts.verify(**c)
    assert np.array_equal(got[0].reshape(-1, 3, 2), np.broadcast_to(few[0], (n // 3, 3, 2))) and np.array_equal(got[1].reshape(-1, 3), np.broadcast_to(few[1], (n // 3, 3)))
    check(case(1, 1, 1024 * 4096))
    for requests, vocab, message in ((n + 1, 2, "bad sizes"), (1, 1024 * 4096 + 1, "vocabulary")):
        i32 = dict(dtype=torch.int32, device=DEV)
        with pytest.raises(ops().KernelError, match=message):
            ops().verify_drafts(torch.zeros((requests, vocab), device=DEV), torch.zeros((requests, 0), **i32), torch.ones(requests, device=DEV), torch.zeros((requests, 1), device=DEV),
                                torch.zeros((requests, 1), **i32), torch.zeros(requests, **i32))
