"""Passes of more than 96 rows whose columns are shared by a cluster, and shorter ones on both sides of the line: every type, gated
pairs, groups."""
import numpy as np
import pytest

import expert_ops_oracle as eo
from graph_util import captured_kernels
from test_gpu_mxfp4 import Held, coded, device, tt

pytestmark = pytest.mark.gpu

# (rows, R, C, activation, groups or None, blocks of the launch)
SHAPES = [(97, 60, 9760, None, None, 8), (427, 18, 9408, None, None, 32), (300, 100, 9760, "silu", None, 48), (120, 70, 12000, "gelu_tanh", None, 16),
          (300, 100, 8032, None, None, 32), (97, 1, 8032, None, None, 16), (311, 60, 9504, None, [120, 0, 191], None),
          (500, 30, 12832, "silu", [0, 250, 250], None)]


@pytest.mark.parametrize("n,R,C,activation,groups,blocks", SHAPES)
@pytest.mark.parametrize("y_dtype,y_pad", [("bf16", 0), ("f32", 3), ("f16", 8)])
def test_long_passes_shared_by_clusters(n, R, C, activation, groups, blocks, y_dtype, y_pad):
    import torch
    counts = groups or [n]
    held = Held(R + C, len(counts), R, C, activation)
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    codes, scales, xv = coded(n, n, C)
    off, y = device(offsets), torch.full((n + 1, R + y_pad), 55.0, dtype=tt(y_dtype), device="cuda")
    torch.cuda.synchronize()
    to = dict(y_dtype=y_dtype, y_row_stride=R + y_pad)

    def call(stream=0):
        args = (codes.data_ptr(), scales.data_ptr())
        rc = (held.handle.experts(*args, off.data_ptr(), n, y.data_ptr(), stream=stream, **to) if groups
              else held.handle.matmul(*args, n, y.data_ptr(), stream=stream, **to))
        assert rc == 0
    call()
    torch.cuda.synchronize()
    assert held.handle.status() == 0
    got = y.double().cpu().numpy()
    assert (got[n:] == 55.0).all() and (got[:, R:] == 55.0).all()
    for e in range(len(counts)):
        b, t = offsets[e], offsets[e + 1]
        if t > b:
            want, err = held.want(xv[b:t], e)
            eo.close(got[b:t, :R], want, err, y_dtype, f"group {e}")
    (name, grid), = captured_kernels(call)
    assert "ELb0EEEv" in name
    if blocks:
        assert grid[0] == blocks
    else:                                                # as many units as the groups may need, a multiple of their cluster
        assert grid[0] > (n // 96 + len(counts)) * ((R * (2 if activation else 1) + 127) // 128)
