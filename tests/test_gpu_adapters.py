"""Low-rank adapters of many requests against the formula in 64 bits.

How far a result may be off, with s the sum of the absolute values that its formula adds up (|base| + scale |B| |A| |x|):
  32-bit sums of at most width + rank + 4 terms, in whatever order, are off by at most that many steps of 2^-24 relative to s;
  a result stored as bfloat16 is off by 2^-8 of itself.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def ops():
    from geneinfer_amd.kernels import ops as o
    return o


def make(n, width, columns, rank, adapters, *, dtype=BF16, w_dtype=None, slices=None, seed=0, ids="mixed", base=F32):
    g = torch.Generator().manual_seed(seed + n + 31 * width + 17 * columns + rank)
    S = 1 if slices is None else len(slices)
    if ids == "mixed":                                        # every row its own draw, some without an adapter
        who = torch.randint(-1, adapters, (n,), generator=g)
    elif ids == "runs":                                       # requests of several rows, one after the other
        who = torch.repeat_interleave(torch.randint(-1, adapters, (n,), generator=g), torch.randint(1, 40, (n,), generator=g))[:n]
    else:
        who = torch.full((n,), ids)
    w_dtype = w_dtype or dtype
    return dict(x=torch.randn(n, width, generator=g).to(dtype).to(DEV), a=(torch.randn(adapters, S * rank, width, generator=g) / width ** 0.5).to(w_dtype).to(DEV),
                b=torch.randn(adapters, columns, rank, generator=g).to(w_dtype).to(DEV), ids=who.int().to(DEV), scales=(torch.rand(adapters, generator=g) + 0.5).to(DEV),
                base=torch.randn(n, columns, generator=g).to(base).to(DEV), slices=slices)


def formula(x, a, b, ids, scales, base, slices, absolute=False):
    f = (lambda t: t.double().abs()) if absolute else (lambda t: t.double())
    out, rank = f(base).clone(), b.shape[2]
    slices = slices or (b.shape[1],)
    for e in range(a.shape[0]):
        rows = (ids == e).nonzero()[:, 0]
        start = 0
        for s, c in enumerate(slices):
            t = f(x[rows]) @ f(a[e, s * rank:(s + 1) * rank]).t()
            out[rows, start:start + c] += (1.0 if scales is None else float(scales[e])) * (t @ f(b[e, start:start + c]).t())
            start += c
    return out


def assert_right(got, c):
    args = {k: c[k] for k in ("x", "a", "b", "ids", "scales", "base", "slices")}
    want, size = formula(**args), formula(**args, absolute=True)
    steps = (c["x"].shape[1] + c["b"].shape[2] + 4) * 2.0 ** -24
    bound = size * steps
    if got.dtype == BF16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    off = (got.double() - want).abs()
    assert bool((off <= bound + 1e-38).all()), f"off by up to {float((off / (bound + 1e-38)).max()):.3f} of what rounding explains"


def run(c, result=F32, in_place=False):
    n, columns = c["base"].shape
    room = torch.full((n + 2, columns + 5), -77.0, dtype=result, device=DEV)
    out = room[1:-1, 2:2 + columns]
    if in_place:
        out.copy_(c["base"])
    got = ops().adapters_add(c["x"], c["a"], c["b"], c["ids"], out, scales=c["scales"], base=None if in_place else c["base"], slices=c["slices"])
    assert got is out
    rim = room.clone()
    rim[1:-1, 2:2 + columns] = -77.0
    assert (rim == -77.0).all()
    return out.clone()


SIZES = [(1, 1, 1, 1, 1), (1, 8, 16, 8, 2), (1, 2048, 2048, 16, 3), (3, 65, 33, 5, 2), (7, 256, 129, 16, 8), (16, 512, 512, 32, 4), (17, 264, 200, 24, 5), (33, 520, 264, 1, 33), (64, 1024, 1000, 64, 70),
         (65, 1000, 72, 12, 3), (100, 2049, 130, 7, 9), (129, 640, 384, 128, 3), (250, 328, 520, 130, 4), (515, 4096, 256, 16, 6), (70, 72, 4104, 40, 2), (300, 31, 31, 31, 31),
         (130, 96, 80, 256, 2), (20, 96, 80, 256, 2), (200, 100, 50, 225, 9), (1200, 1536, 1100, 48, 3),
         (600, 328, 520, 128, 4), (530, 96, 80, 256, 2), (520, 264, 200, 24, 5), (40, 264, 201, 4, 9), (7, 1032, 96, 12, 7), (3, 72, 600, 6, 2), (2, 4096, 512, 10, 2), (90, 136, 64, 1, 3), (900, 264, 2048, 12, 4), (700, 520, 1024, 44, 3), (800, 128, 512, 10, 2), (1600, 520, 2100, 104, 3), (1600, 264, 2100, 72, 3), (1700, 264, 2048, 52, 4), (1700, 264, 2048, 36, 4), (1025, 1000, 72, 40, 1100)]


@pytest.mark.parametrize("n,width,columns,rank,adapters", SIZES)
@pytest.mark.parametrize("dtypes", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
def test_against_64_bits(n, width, columns, rank, adapters, dtypes):
    for ids in ("mixed", "runs"):
        c = make(n, width, columns, rank, adapters, dtype=dtypes[0], w_dtype=dtypes[1], ids=ids)
        assert_right(run(c), c)


@pytest.mark.parametrize("n", [1, 5, 64, 90, 300, 560])
@pytest.mark.parametrize("base", [F32, BF16])
@pytest.mark.parametrize("result", [F32, BF16])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_dtypes_of_base_and_result_and_in_place(n, base, result, dtype):
    c = make(n, 264, 296, 16, 4, dtype=dtype, base=base, ids="runs")
    apart = run(c, result)
    assert_right(apart, c)
    if base == result:
        assert torch.equal(run(c, result, in_place=True), apart)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 9, 200, 570])
@pytest.mark.parametrize("slices,rank", [((256, 64, 64), 16), ((100, 29), 8), ((1, 500, 3, 8), 5), ((40, 40, 40, 40), 64)])
def test_packed_projections(n, slices, rank, dtype):
    for scales in (True, False):
        c = make(n, 384, sum(slices), rank, 3, slices=slices, dtype=dtype, ids="runs")
        c["scales"] = c["scales"] if scales else None
        assert_right(run(c, dtype), c)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 70, 260, 515])
def test_rows_without_an_adapter_are_the_base(n, dtype):
    c = make(n, 128, 200, 16, 4, dtype=dtype, ids=-1)
    c["x"][:] = float("nan")                                  # (nothing of theirs is read into a result)
    assert torch.equal(run(c), c["base"])
    c["ids"][:] = 4
    assert torch.equal(run(c), c["base"])
    c["ids"][::2] = torch.iinfo(torch.int32).max
    c["ids"][1::2] = torch.iinfo(torch.int32).min
    assert torch.equal(run(c), c["base"])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_row_of_no_numbers_stays_its_own(dtype):
    """NaN and infinities of one request's rows, or of an adapter that others do not take, reach no other row."""
    for n in (8, 96, 256, 600):
        c = make(n, 256, 144, 16, 4, dtype=dtype, ids="mixed")
        c["ids"][:4] = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
        clean = run(c)
        bad = dict(c, x=c["x"].clone(), a=c["a"].clone(), b=c["b"].clone())
        bad["x"][0] = float("nan")
        bad["a"][1, 3, 7] = float("inf")
        bad["b"][2, 5] = float("nan")
        got, ids = run(bad), c["ids"]
        same = (ids != 1) & (ids != 2)
        same[0] = False
        assert torch.equal(got[same], clean[same])
        assert got[0].isnan().all() and not got[ids == 1].isfinite().any() and got[ids == 2][:, 5].isnan().all()
        others = got[ids == 2]
        assert torch.equal(torch.cat([others[:, :5], others[:, 6:]], 1), torch.cat([clean[ids == 2][:, :5], clean[ids == 2][:, 6:]], 1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rank", [5, 8, 20, 24, 36, 40, 72, 96, 136, 200])
def test_a_row_of_no_numbers_stays_its_own_at_every_rank(rank, dtype):
    """The ranks' places behind the last, which the products run over, hold nothing of the rows beside."""
    for n in (90, 1600):
        c = make(n, 128, 2048, rank, 2, dtype=dtype, ids=0)
        clean = run(c)
        for bad in (float("nan"), float("inf")):
            other = dict(c, x=c["x"].clone())
            other["x"][3::5] = bad
            got = run(other)
            whole = torch.ones(n, dtype=torch.bool, device=DEV)
            whole[3::5] = False
            assert torch.equal(got[whole], clean[whole])
            assert not got[~whole].isfinite().any()


@pytest.mark.parametrize("n", [1, 20, 600])
def test_sums_that_bfloat16_cannot_hold(n):
    """Sums A x at the end of 32 bits, beyond bfloat16's, stay the numbers that they are, and infinite ones infinite."""
    c = make(n, 64, 48, 8, 1, dtype=BF16, ids=0)
    c["scales"] = None
    c["x"].zero_()
    c["x"][:, 0] = 2.0 ** 127
    c["a"].zero_()
    c["a"][0, :, 0], c["a"][0, :, 1] = 1.9921875, 2.0 ** -8   # (together 1.998 * 2^127; the most that bfloat16 has is 1.9922 * 2^127)
    c["x"][:, 1] = 2.0 ** 127 * 1.5
    c["b"].fill_(2.0 ** -120)
    assert_right(run(c), c)
    c["x"][::2, 2], c["a"][0, :, 2] = float("inf"), 1.0
    got = run(c)
    assert bool((got[::2] == float("inf")).all()) and bool(got[1::2].isfinite().all())


@pytest.mark.parametrize("width,rank", [(256, 16), (1000, 24), (77, 5), (4096, 64)])
@pytest.mark.parametrize("w_dtype", [F32, BF16])
def test_a_32_bit_row_has_the_same_bits_in_every_batch(w_dtype, width, rank):
    c = make(300, width, 328, rank, 5, dtype=F32, w_dtype=w_dtype, ids="runs")
    whole = run(c)
    for rows in (slice(0, 1), slice(17, 18), slice(299, 300), slice(5, 25), slice(100, 165), slice(3, 259)):
        part = dict(c, x=c["x"][rows], ids=c["ids"][rows].clone(), base=c["base"][rows])
        assert torch.equal(run(part), whole[rows])
    order = torch.randperm(300, generator=torch.Generator().manual_seed(1)).to(DEV)
    assert torch.equal(run(dict(c, x=c["x"][order], ids=c["ids"][order], base=c["base"][order])), whole[order])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_places(dtype):
    for n in (5, 150, 530):
        c = make(n, 192, 96, 16, 3, dtype=dtype, ids="runs")
        wide = torch.full((n, 400), 9.0, dtype=dtype, device=DEV)
        for first in (0, 3, 8):                               # rows that begin at 16 bytes and that do not
            part = wide[:, first:first + 192]
            part.copy_(c["x"])
            assert_right(run(dict(c, x=part)), c)
        odd = torch.empty((n, 193), dtype=dtype, device=DEV)[:, :192]
        odd.copy_(c["x"])
        assert_right(run(dict(c, x=odd)), c)
        flat = torch.empty(c["a"].numel() + 1, dtype=dtype, device=DEV)[1:].view(c["a"].shape)
        flat.copy_(c["a"])
        up = torch.empty(c["b"].numel() + 1, dtype=dtype, device=DEV)[1:].view(c["b"].shape)
        up.copy_(c["b"])
        assert_right(run(dict(c, a=flat, b=up)), c)
        base = torch.empty((n, 99), device=DEV)[:, 1:97]
        base.copy_(c["base"])
        assert_right(run(dict(c, base=base)), c)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_single_row_of_a_buffer_whose_rows_are_far_apart(dtype):
    """Rows may be at most 2^23 numbers apart; one row is apart from none."""
    c = make(1, 128, 96, 16, 3, dtype=dtype, ids=1)
    apart = 2 ** 23 + 64
    out, base = torch.zeros((2, apart), device=DEV)[1:, 7:103], torch.zeros((2, apart), device=DEV)[1:, 1:97]
    base.copy_(c["base"])
    assert_right(ops().adapters_add(c["x"], c["a"], c["b"], c["ids"], out, scales=c["scales"], base=base), c)
    two = make(2, 128, 96, 16, 3, dtype=dtype, ids=1)
    with pytest.raises(ops().KernelError, match="numbers apart"):
        ops().adapters_add(two["x"], two["a"], two["b"], two["ids"], torch.zeros((2, apart), device=DEV)[:, :96], scales=two["scales"], base=two["base"])


def test_captured_and_replayed_with_other_requests():
    for n in (6, 140, 600):
        cs = [make(n, 512, 640, 16, 4, seed=s, ids="runs") for s in range(3)]
        held = {k: v.clone() if torch.is_tensor(v) else v for k, v in cs[0].items()}
        out = torch.empty_like(held["base"])

        def call():
            ops().adapters_add(held["x"], held["a"], held["b"], held["ids"], out, scales=held["scales"], base=held["base"])

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for c in (*cs, *cs):
            for k, v in c.items():
                if torch.is_tensor(v):
                    held[k].copy_(v)
            graph.replay()
            assert torch.equal(out, run(c))


def test_two_streams_at_once():
    cs = [make(n, 1024, 512, 32, 3, seed=n, ids="runs") for n in (200, 700)]
    want = [run(c) for c in cs]
    outs, streams = [torch.empty_like(c["base"]) for c in cs], [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, out, s in zip(cs, outs, streams):
            with torch.cuda.stream(s):
                ops().adapters_add(c["x"], c["a"], c["b"], c["ids"], out, scales=c["scales"], base=c["base"])
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)


def test_offsets_beyond_32_bits():
    """Numbers of out, and of the adapters' matrices, beyond 2^31."""
    n, width, columns, rank = 70000, 64, 32768, 8
    c = make(n, width, 96, rank, 3, ids="runs")
    out = torch.zeros((n, columns), dtype=BF16, device=DEV)   # 2.3e9 numbers
    got = ops().adapters_add(c["x"], c["a"], c["b"], c["ids"], out[:, -96:], scales=c["scales"], base=c["base"])
    assert_right(got, c)
    assert (out[-1, :-96] == 0).all()
    del out, got
    many = 2 ** 31 // (16 * 8192) + 2
    a = torch.zeros((many, 16, 8192), dtype=BF16, device=DEV)
    b = torch.zeros((many, 40, 16), dtype=BF16, device=DEV)
    for n in (3, 130, 520):
        c = make(n, 8192, 40, 16, 3, ids="mixed")
        place = torch.tensor([0, many // 2, many - 1], device=DEV)
        a[place], b[place] = c["a"], c["b"]
        scales = torch.zeros(many, device=DEV)
        scales[place] = c["scales"]
        ids = torch.where(c["ids"] >= 0, place[c["ids"].clamp_min(0).long()].int(), c["ids"])
        out = ops().adapters_add(c["x"], a, b, ids, torch.empty((n, 40), device=DEV), scales=scales, base=c["base"])
        assert_right(out, c)


@pytest.mark.parametrize("result", [F32, BF16])
@pytest.mark.parametrize("n", [1, 70, 600, 1500])
@pytest.mark.parametrize("columns,slices", [(65, None), (66, None), (67, None), (515, None), (2049, None), (193, (65, 128)), (262, (66, 67, 129)), (1031, (513, 4, 514))])
def test_columns_that_are_no_fours(columns, slices, n, result):
    """One to three columns behind whole blocks, onto base elsewhere and onto base itself; the rows begin at every place."""
    for dtype in (BF16, F32):
        c = make(n, 136, columns, 16, 3, dtype=dtype, ids="runs", base=result, slices=slices)
        apart = run(c, result)
        assert_right(apart, c)
        assert torch.equal(run(c, result, in_place=True), apart)


def test_the_most_rows_and_one_more():
    n = 2 ** 20
    for runs in ("mixed", "runs"):
        c = make(n, 8, 8, 8, 5, ids=runs)
        assert_right(run(c), c)
    x, ids, out = torch.zeros((n + 1, 8), dtype=BF16, device=DEV), torch.zeros(n + 1, dtype=torch.int32, device=DEV), torch.zeros((n + 1, 8), device=DEV)
    with pytest.raises(ops().KernelError, match="too many"):
        ops().adapters_add(x, c["a"], c["b"], ids, out)


def test_the_widest_rows():
    for n in (2, 513):
        c = make(n, 2 ** 16 + 8, 16, 8, 2, ids="mixed")
        assert_right(run(c), c)
    x, a, b = (torch.zeros(shape, dtype=BF16, device=DEV) for shape in ((1, 2 ** 24 + 8), (1, 8, 2 ** 24 + 8), (1, 8, 8)))
    with pytest.raises(ops().KernelError, match="too many"):
        ops().adapters_add(x, a, b, torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros((1, 8), device=DEV))
    c = make(2, 2 ** 24, 8, 8, 1, ids=0)
    assert_right(run(c), c)


@pytest.mark.parametrize("result", [F32, BF16])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 40, 300, 600])
def test_beside_the_shared_projection(n, dtype, result):
    from geneinfer_amd.parts.linear import RowAdapters, linear
    c = make(n, 512, 384, 16, 5, dtype=dtype, ids="runs")
    weight = (torch.randn(384, 512, generator=torch.Generator().manual_seed(n)) / 512 ** 0.5).to(dtype).to(DEV)
    beside = RowAdapters(c["a"], c["b"], c["ids"], c["scales"])
    got = linear(c["x"], weight, torch.empty((n, 384), dtype=result, device=DEV), adapters=beside)
    c["base"] = c["x"].double() @ weight.double().t()
    size = formula(*(c[k] for k in ("x", "a", "b", "ids", "scales")), c["x"].double().abs() @ weight.double().abs().t(), None, absolute=True)
    want = formula(**c)
    bound = size * ((2 * 512 + 16 + 8) * 2.0 ** -24)
    if result == BF16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    assert bool(((got.double() - want).abs() <= bound).all())
    if result == F32:                                         # onto rows that are there
        there = torch.randn(n, 384, generator=torch.Generator().manual_seed(3)).to(DEV)
        onto = linear(c["x"], weight, there.clone(), accumulate=True, adapters=beside)
        assert bool(((onto.double() - there.double() - want).abs() <= bound + 4 * (there.double().abs() + want.abs()) * 2.0 ** -24).all())


def test_adapted_heads_feed_the_judgement_of_drafts():
    """The two as a server uses them: every request's rows through the head with its own adapter, its drafts judged by the logits."""
    import numpy as np
    import plain_drafts
    from geneinfer_amd.parts.linear import RowAdapters, linear
    R, K, width, vocab = 6, 3, 256, 3001
    g = torch.Generator().manual_seed(4)
    c = make(R * (K + 1), width, vocab, 16, 4, seed=4)
    c["ids"] = torch.repeat_interleave(torch.tensor([0, 3, -1, 1, 1, 2]), K + 1).int().to(DEV)
    head = (torch.randn(vocab, width, generator=g) * 3 / width ** 0.5).to(BF16).to(DEV)
    logits = linear(c["x"], head, torch.empty((R * (K + 1), vocab), device=DEV), adapters=RowAdapters(c["a"], c["b"], c["ids"], c["scales"]))
    c["base"] = c["x"].double() @ head.double().t()
    assert float((logits.double() - formula(**c)).abs().max()) < 1e-3
    drafter = logits.view(R, K + 1, vocab)[:, :K] + 0.3 * torch.randn(R, K, vocab, generator=g).to(DEV)
    drafts, uniform = drafter.argmax(-1).int(), torch.rand(R, K + 1, generator=g).to(DEV)
    temperature = torch.tensor([0.7, 0.0, 1.0, 0.7, 0.0, 1.2], device=DEV)
    tokens, counts = torch.empty((R, K + 1), dtype=torch.int32, device=DEV), torch.empty(R, dtype=torch.int32, device=DEV)
    ops().verify_drafts(logits, drafts, temperature, uniform, tokens, counts, draft_logits=drafter)
    want = plain_drafts.verify(logits.cpu().numpy(), drafts.cpu().numpy(), temperature.cpu().numpy(), uniform.cpu().numpy(), drafter.cpu().numpy())
    assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(counts.cpu().numpy(), want[1])
