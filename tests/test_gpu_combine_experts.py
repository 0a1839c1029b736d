"""The weighted combine of experts' rows against 64 bits: types, odd widths and strides, missing rows, long rows."""
import importlib

import numpy as np
import pytest

import expert_ops_oracle as eo

pytestmark = pytest.mark.gpu
ex = importlib.import_module("salt-core_b200.experts")
TYPES = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def check(tokens, topk, cols, dtype="f32", y_dtype="f32", pad=0, y_pad=0, index=True, shift=0, lost=0.0, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = tokens * topk
    flat = torch.randn(n * (cols + pad) + shift, device="cuda", generator=g).to(getattr(torch, TYPES[dtype]))
    rows = flat[shift:].view(n, cols + pad)
    w = torch.rand(tokens, topk, device="cuda", generator=g)
    idx = torch.randperm(n, device="cuda", generator=g).to(torch.int32)
    idx[torch.rand(n, device="cuda", generator=g) < lost] = -1
    if n > 3 and lost:
        idx[1], idx[3] = n, 2 ** 31 - 1                  # beyond the rows: adds nothing
    y = torch.full((tokens, cols + y_pad), 55.0, dtype=getattr(torch, TYPES[y_dtype]), device="cuda")
    torch.cuda.synchronize()
    assert ex.combine(rows.data_ptr(), n, cols, idx.data_ptr() if index else 0, w.data_ptr(), tokens, topk, y.data_ptr(), dtype=dtype,
                      y_dtype=y_dtype, row_stride=cols + pad, y_row_stride=cols + y_pad) == 0
    torch.cuda.synchronize()
    r, wn = rows[:, :cols].double().cpu().numpy(), w.double().cpu().numpy()
    i = idx.cpu().numpy().reshape(tokens, topk) if index else np.arange(n).reshape(tokens, topk)
    ok = (i >= 0) & (i < n)
    terms = np.where(ok, wn, 0.0)[:, :, None] * r[np.where(ok, i, 0)]
    # topk fused steps, each rounding at most half a unit of what has been added
    eo.close(y[:, :cols].double().cpu().numpy(), terms.sum(axis=1), topk * 2.0 ** -24 * np.abs(terms).sum(axis=1), y_dtype)
    assert (y[:, cols:] == 55.0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("y_dtype", list(TYPES))
@pytest.mark.parametrize("cols", [1, 8, 37, 1024, 2816, 1032])
def test_types_and_widths(dtype, y_dtype, cols):
    check(13, 4, cols, dtype, y_dtype, seed=cols)


@pytest.mark.parametrize("topk", [1, 2, 3, 8, 31, 32])
def test_topk(topk):
    check(7, topk, 520, "bf16", "bf16", seed=topk)


@pytest.mark.parametrize("pad,y_pad,shift", [(8, 0, 0), (3, 0, 0), (0, 5, 0), (0, 0, 1), (8, 16, 8), (4, 0, 4)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_alignment(pad, y_pad, shift, dtype):
    check(5, 3, 64, dtype, dtype, pad, y_pad, shift=shift, seed=pad + y_pad)


@pytest.mark.parametrize("index", [False, True])
def test_missing_rows(index):
    check(40, 6, 200, "f16", "f32", index=index, lost=0.4 if index else 0.0)
    check(9, 4, 64, lost=1.0)


def test_values_that_are_not_numbers():
    """An infinity or NaN in a row reaches the tokens that use it, and no others; a missing one reaches none."""
    import torch
    rows = torch.ones(6, 16, device="cuda")
    rows[1, 2], rows[4] = torch.inf, torch.nan
    idx = torch.tensor([0, 1, 2, -1, 3, 5], dtype=torch.int32, device="cuda")
    w = torch.full((6,), 0.5, device="cuda")
    y = torch.empty(3, 16, device="cuda")
    assert ex.combine(rows.data_ptr(), 6, 16, idx.data_ptr(), w.data_ptr(), 3, 2, y.data_ptr()) == 0
    want = torch.ones(3, 16)
    want[0, 2], want[1] = torch.inf, 0.5
    assert torch.equal(y.cpu(), want)


def test_many_tokens():
    check(70001, 2, 24, "bf16", "bf16", seed=9)


def test_offsets_beyond_32_bits():
    """Row 2^21 + 5 of rows 1024 + 8 elements apart: an element offset above 2^31."""
    import torch
    stride, n = 1032, (1 << 21) + 6
    rows = torch.zeros(n * stride, dtype=torch.bfloat16, device="cuda")
    at = n - 1
    rows[at * stride:at * stride + 64] = torch.arange(64, device="cuda").to(torch.bfloat16)
    idx = torch.tensor([at, 0], dtype=torch.int32, device="cuda")
    w = torch.ones(2, device="cuda")
    y = torch.empty(1, 64, device="cuda")
    assert ex.combine(rows.data_ptr(), n, 64, idx.data_ptr(), w.data_ptr(), 1, 2, y.data_ptr(), dtype="bf16", row_stride=stride) == 0
    assert torch.equal(y[0].cpu(), torch.arange(64.0))


def test_no_rows():
    """Tokens none of whose rows exist are zeros, also where there are no rows at all."""
    import torch
    for cols in (64, 37):
        y = torch.full((3, cols), 55.0, device="cuda")
        idx = torch.full((6,), -1, dtype=torch.int32, device="cuda")
        w = torch.ones(6, device="cuda")
        assert ex.combine(0, 0, cols, idx.data_ptr(), w.data_ptr(), 3, 2, y.data_ptr()) == 0
        assert not y.any()
        y.fill_(55.0)
        assert ex.combine(0, 0, cols, 0, w.data_ptr(), 3, 2, y.data_ptr()) == 0
        assert not y.any()
