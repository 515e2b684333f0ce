"""Judging drafts and adding adapters refuse operands that their kernels do not take, before anything is launched (no GPU needed)."""
import pytest
import torch

from geneinfer_amd.kernels import ops


def verify_args(n=3, k=2, vocab=50, rows=9):
    return dict(logits=torch.zeros(rows, vocab), drafts=torch.zeros((n, k), dtype=torch.int32), temperature=torch.ones(n), uniform=torch.zeros(n, k + 1),
                tokens=torch.zeros((n, k + 1), dtype=torch.int32), counts=torch.zeros(n, dtype=torch.int32))


@pytest.mark.parametrize("change,message", [
    (dict(logits=torch.zeros(9, 50, dtype=torch.bfloat16)), "logits"), (dict(logits=torch.zeros(9, 100)[:, ::2]), "logits"), (dict(logits=torch.zeros(450)), "logits"),
    (dict(logits=torch.zeros(9, 0)), "logits"), (dict(logits=torch.zeros(8, 50)), "9 rows"), (dict(drafts=torch.zeros((3, 2), dtype=torch.int64)), "drafts"),
    (dict(drafts=torch.zeros((2, 3), dtype=torch.int32).t()), "drafts"), (dict(temperature=torch.ones(2)), "temperature"), (dict(temperature=torch.ones(3, dtype=torch.float64)), "temperature"),
    (dict(uniform=torch.zeros(3, 2)), "uniform"), (dict(tokens=torch.zeros((3, 2), dtype=torch.int32)), "tokens"), (dict(counts=torch.zeros(3, dtype=torch.int64)), "counts"),
    (dict(n_drafts=torch.zeros(2, dtype=torch.int32)), "n_drafts"), (dict(first_row=torch.zeros(3)), "first_row"), (dict(draft_logits=torch.zeros(3, 2, 49)), "draft_logits"),
    (dict(draft_logits=torch.zeros(3, 2, 50, dtype=torch.bfloat16)), "draft_logits"), (dict(draft_logits=torch.zeros(3, 50, 2).transpose(1, 2)), "draft_logits"),
    (dict(drafts=torch.zeros((3, 65), dtype=torch.int32)), "at most 64"), ({}, "device memory"),
])
def test_verify_refuses(change, message):
    with pytest.raises(ops.KernelError, match=message):
        ops.verify_drafts(**{**verify_args(), **change})


def test_verify_without_rows():
    with pytest.raises(ops.KernelError, match="no rows"):
        ops.verify_drafts(**{**verify_args(), "logits": torch.zeros(0, 50), "first_row": torch.zeros(3, dtype=torch.int32)})


def adapter_args(n=5, width=16, columns=12, rank=4, adapters=3, slices=1):
    return dict(x=torch.zeros(n, width), a=torch.zeros(adapters, rank * slices, width), b=torch.zeros(adapters, columns, rank), ids=torch.zeros(n, dtype=torch.int32), out=torch.zeros(n, columns))


@pytest.mark.parametrize("change,message", [
    (dict(x=torch.zeros(5, 15)), "do not fit"), (dict(x=torch.zeros(80)), "needed"), (dict(x=torch.zeros(5, 16, dtype=torch.float16)), "dtype"),
    (dict(x=torch.zeros(5, 32)[:, ::2]), "unit inner stride"), (dict(x=torch.zeros(1, 16).expand(5, 16)), "overlap"), (dict(out=torch.zeros(5, 11)), "do not fit"),
    (dict(out=torch.zeros(1, 12).expand(5, 12)), "overlap"), (dict(base=torch.zeros(4, 12)), "do not fit"), (dict(base=torch.zeros(5, 12, dtype=torch.float64)), "dtype"),
    (dict(a=torch.zeros(3, 16, 4).transpose(1, 2)), "contiguous"), (dict(a=torch.zeros(3, 4, 16, dtype=torch.bfloat16)), "one dtype"), (dict(b=torch.zeros(2, 12, 4)), "do not fit"),
    (dict(ids=torch.zeros(5, dtype=torch.int64)), "ids"), (dict(ids=torch.zeros(4, dtype=torch.int32)), "ids"), (dict(scales=torch.ones(2)), "scales"),
    (dict(scales=torch.ones(3, dtype=torch.bfloat16)), "scales"), (dict(slices=(6, 5)), "slices"), (dict(slices=(12, 0)), "slices"), (dict(slices=()), "slices"),
    (dict(slices=(3, 3, 2, 2, 2)), "slices"), (dict(slices=(6, 6)), "do not fit"), (dict(a=torch.zeros(3, 0, 16), b=torch.zeros(3, 12, 0)), "no entries"),
    (dict(a=torch.zeros(3, 257, 16), b=torch.zeros(3, 12, 257)), "at most 256"), ({}, "device memory"),
])
def test_adapters_refuse(change, message):
    with pytest.raises(ops.KernelError, match=message):
        ops.adapters_add(**{**adapter_args(), **change})


def test_base_and_out_at_one_place_must_be_the_same():
    args = adapter_args()
    room = torch.zeros(5, 24)
    for base, out in ((room.view(10, 12)[:5], room[:, :12]), (room.view(torch.bfloat16)[:, :12], room[:, :12])):
        with pytest.raises(ops.KernelError, match="same place"):
            ops.adapters_add(**{**args, "base": base, "out": out})


def test_x_and_out_at_one_place():
    args = adapter_args(columns=16)
    with pytest.raises(ops.KernelError, match="x and out begin at the same place"):
        ops.adapters_add(**{**args, "out": args["x"]})
    room = torch.zeros(5, 32)                                 # beside one another in one buffer they share nothing
    with pytest.raises(ops.KernelError, match="device memory"):
        ops.adapters_add(**{**args, "x": room[:, :16], "out": room[:, 16:]})


def test_adapters_of_no_rows_change_nothing():
    args = adapter_args(n=0)
    assert ops.adapters_add(**args) is args["out"]


def test_a_gated_product_and_rounded_sums_take_no_adapters():
    from geneinfer_amd.parts.linear import RowAdapters, linear
    args = adapter_args()
    adapters = RowAdapters(args["a"], args["b"], args["ids"])
    with pytest.raises(ops.KernelError, match="gated"):
        linear(args["x"], torch.zeros(12, 16), args["out"], gated=True, adapters=adapters)
    with pytest.raises(ops.KernelError, match="float32 rows only"):
        linear(args["x"], torch.zeros(12, 16), args["out"].bfloat16(), accumulate=True, adapters=adapters)
