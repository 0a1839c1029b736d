"""Calls that the documentation allows and that leave an argument out."""
import importlib

import pytest

import expert_ops_oracle as eo

pytestmark = pytest.mark.gpu
ex = importlib.import_module("salt-core_b200.experts")


@pytest.mark.parametrize("div", [0, -3, 7])
def test_the_divisor_is_not_read_without_an_index(div):
    import numpy as np
    import torch
    n, cols = 5, 96
    x = torch.randn(n, cols, device="cuda")
    codes = torch.zeros(n, cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(n, eo.scale_pitch(cols), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert ex.quantize(x.data_ptr(), n, cols, codes.data_ptr(), scales.data_ptr(), index_div=div) == 0
    torch.cuda.synchronize()
    code, byte = eo.mx_quantize(x.double().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), eo.mx_pack(code)) and np.array_equal(scales[:, :cols // 32].cpu().numpy(), byte)
