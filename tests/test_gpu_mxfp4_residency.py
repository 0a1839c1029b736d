"""Blocks of an MXFP4 product that wait for one another hold tensor memory while they do: which of them can share an SM follows from
the shared memory that they ask for, read from a capture."""
import pytest

from graph_util import captured_launches
from test_gpu_mxfp4 import Held, acts, check_matmul

pytestmark = pytest.mark.gpu
SM_BYTES, OWN_BYTES = 228 * 1024, 10 * 1024      # of an SM; of a block beside its dynamic part (tables 9 KB, the system 1 KB)


def launch(held, n, R, C):
    import torch
    codes, scales, _ = acts(n, n, C)
    y = torch.empty(n, R, device="cuda")

    def call(stream=0):
        assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr(), stream=stream) == 0
    (name, grid, shared), = captured_launches(call)
    return name, grid[0], shared


def test_waiting_blocks_do_not_share_tensor_memory():
    """Two blocks of pairs, or of clusters that take all of tensor memory, never share an SM, nor does one of them with a block of a
    cluster that takes half of it (two of those may).  Shapes whose blocks ask for little."""
    pairs, wide, halves = [], [], []
    for n, R, C in ((437, 3386, 1504), (218, 6679, 1536), (770, 1300, 5056)):
        held = Held(R + C, 1, R, C)
        name, grid, shared = launch(held, n, R, C)
        assert "ELb1EEEv" in name
        pairs.append(shared)
    for n, R, C in ((97, 60, 9760), (427, 18, 9408)):
        held = Held(R + C, 1, R, C)
        name, grid, shared = launch(held, n, R, C)
        passes = grid // 8                               # one row tile, clusters of eight
        assert "ELb0EEEv" in name and grid % 8 == 0 and passes * 96 < n
        wide.append(shared)
        check_matmul(held, n, R, C)
    for n, R, C in ((1, 128, 2048), (221, 167, 3392), (233, 429, 1888), (20, 500, 2048)):
        held = Held(R + C, 1, R, C)
        name, grid, shared = launch(held, n, R, C)
        assert "ELb0EEEv" in name and grid > (R + 127) // 128
        halves.append(shared)
        check_matmul(held, n, R, C)
    least = min(pairs + wide) + OWN_BYTES
    assert 2 * least > SM_BYTES
    assert least + min(halves) + OWN_BYTES > SM_BYTES
