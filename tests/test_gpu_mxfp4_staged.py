"""Long passes with result rows on sixteen bytes, of every type: on pairs of SMs they leave through shared memory, full tiles beside a
last one that is not, so that a block's epilogue takes both ways in turn; on single SMs they do not."""
import numpy as np
import pytest

import expert_ops_oracle as eo
from graph_util import captured_kernels
from test_gpu_mxfp4 import Held, coded, device, tt

pytestmark = pytest.mark.gpu

# (rows, R, C, activation, groups or None, runs on pairs of SMs)
SHAPES = [(1001, 2824, 2848, None, None, True), (1537, 1416, 4000, "gelu_tanh", None, True), (18889, 128, 1408, None, None, False),
          (18889, 64, 1408, "silu", None, False), (2600, 1304, 1568, None, [700, 0, 224, 225, 226, 900, 1, 324], True),
          (2600, 648, 1568, "silu", [3, 2590, 0, 7, 0, 0, 0, 0], True), (14967, 128, 1376, None, [7000, 0, 7967], False)]


@pytest.mark.parametrize("n,R,C,activation,groups,pair", SHAPES)
@pytest.mark.parametrize("y_dtype,y_pad", [("bf16", 0), ("f16", 8), ("f32", 0)])
def test_results_through_shared_memory(n, R, C, activation, groups, pair, y_dtype, y_pad):
    import torch
    counts = groups or [n]
    held = Held(R + C, len(counts), R, C, activation)
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    codes, scales, xv = coded(n, n, C)
    off, y = device(offsets), torch.full((n + 1, R + y_pad), 55.0, dtype=tt(y_dtype), device="cuda")
    assert y.data_ptr() % 16 == 0 and y.stride(0) * y.element_size() % 16 == 0
    torch.cuda.synchronize()
    to = dict(y_dtype=y_dtype, y_row_stride=R + y_pad)

    def call(stream=0):
        args = (codes.data_ptr(), scales.data_ptr())
        rc = (held.handle.experts(*args, off.data_ptr(), n, y.data_ptr(), stream=stream, **to) if groups
              else held.handle.matmul(*args, n, y.data_ptr(), stream=stream, **to))
        assert rc == 0
    for _ in range(3):
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
    (name, _), = captured_kernels(call)
    assert ("ELb1EEEv" in name) == pair
