"""Rows up to the documented width, on sums that are exact in 32 bits, so that every result is compared bit for bit: a block of 32
columns that is skipped, counted twice or scaled by another block's byte shows in it, however long the row."""
import importlib

import numpy as np
import pytest

import expert_ops_oracle as eo
from test_gpu_mxfp4 import device

pytestmark = pytest.mark.gpu
ex = importlib.import_module("salt-core_b200.experts")


def marked_blocks(C):
    """The first and the last blocks of a row, both sides of every border that a share of the row can have among 1, 2, 4 or 8 blocks of a
    cluster, and each step of 64 columns of the last two chunks of 256."""
    blocks, chunks = C // 32, -(-C // 256)
    at = {0, 1, blocks - 1}
    for split in (2, 4, 8):
        share = -(-chunks // split)
        for k in range(share, chunks, share):
            at |= {8 * k - 1, 8 * k}
    at |= set(range(max(0, 8 * (chunks - 2)), blocks))
    return np.array(sorted(b for b in at if 0 <= b < blocks))


@pytest.mark.parametrize("C", [131072, 131040, 40960, 33056, 8192, 2080])
@pytest.mark.parametrize("R,groups", [(40, False), (300, False), (130, True)])
def test_every_block_counts(C, R, groups):
    """A row of weights has four marked blocks, the others are zeros with any scale; activations are dense.  Products are multiples of
    2^-6 (codes of a half, scales down to 2^-2 on both sides) and 128 of them stay below 36 x 128 x 2^4 = 2^16.2: 23 bits."""
    import torch
    rng = np.random.default_rng(C + R)
    E, blocks, marks = (3 if groups else 1), C // 32, marked_blocks(C)
    code, byte = np.zeros((E, R, C), np.uint8), rng.integers(0, 255, (E, R, blocks)).astype(np.uint8)
    turn = rng.permutation(len(marks))
    for e in range(E):
        for r in range(R):
            for j in range(min(4, len(marks))):
                b = marks[turn[(4 * (e * R + r) + j) % len(marks)]]
                code[e, r, 32 * b:32 * b + 32] = rng.integers(0, 16, 32)
                byte[e, r, b] = rng.integers(125, 130)
    values = eo.mx_values(code, np.where((code.reshape(E, R, blocks, 32) == 0).all(axis=3), 127, byte))
    wc, wb = device(eo.mx_pack(code)), device(byte)
    handle = ex.Mxfp4Weights(R, C, E, wc.data_ptr(), wb.data_ptr())
    for n in (1, 20, 130):
        xcode, xbyte = rng.integers(0, 16, (n, C)).astype(np.uint8), rng.integers(125, 130, (n, blocks)).astype(np.uint8)
        held = np.full((n, eo.scale_pitch(C)), 0xff, np.uint8)
        held[:, :blocks] = xbyte
        xc, xs, xv = device(eo.mx_pack(xcode)), device(held), eo.mx_values(xcode, xbyte)
        y = torch.full((n, R), 55.0, device="cuda")
        bounds = [0, n // 3, n // 3, n] if groups else [0, n]
        off = device(np.array(bounds, np.int32))
        torch.cuda.synchronize()
        if groups:
            assert handle.experts(xc.data_ptr(), xs.data_ptr(), off.data_ptr(), n, y.data_ptr()) == 0
        else:
            assert handle.matmul(xc.data_ptr(), xs.data_ptr(), n, y.data_ptr()) == 0
        torch.cuda.synchronize()
        assert handle.status() == 0
        want = np.concatenate([xv[b:t] @ values[e].T for e, (b, t) in enumerate(zip(bounds, bounds[1:]))])
        assert np.array_equal(y.double().cpu().numpy(), want), (n, np.argwhere(y.double().cpu().numpy() != want)[:5])
