"""The activation between the two rows of a gated pair, on gate and up sums that are exact in 32 bits: far on both sides of zero, and
where a block is not a number."""
import importlib

import numpy as np
import pytest

import expert_ops_oracle as eo
from test_gpu_mxfp4 import device, tt

pytestmark = pytest.mark.gpu
ex = importlib.import_module("salt-core_b200.experts")


def pair(seed, R, C, activation, gate_byte, up_byte):
    """A gated pair of random codes whose blocks all have the same scale: every product and partial sum is a multiple of a quarter of
    the scale product below 2^24 of them."""
    rng = np.random.default_rng(seed)
    codes = [rng.integers(0, 16, (1, R, C)).astype(np.uint8) for _ in range(2)]
    bytes_ = [np.full((1, R, C // 32), b, np.uint8) for b in (gate_byte, up_byte)]
    dev = [device(a) for c, b in zip(codes, bytes_) for a in (eo.mx_pack(c), b)]
    handle = ex.Mxfp4Weights(R, C, 1, dev[0].data_ptr(), dev[1].data_ptr(), up_codes=dev[2].data_ptr(), up_scales=dev[3].data_ptr(),
                             activation=activation)
    return handle, codes, bytes_


def rows(seed, n, C):
    rng = np.random.default_rng(seed)
    code = rng.integers(0, 16, (n, C)).astype(np.uint8)
    scale = np.full((n, eo.scale_pitch(C)), 127, np.uint8)
    return device(eo.mx_pack(code)), device(scale), eo.mx_values(code, scale[:, :C // 32])


def act_in_steps(name, g):
    """(value in 64 bits, bound on the error of its evaluation in 32 bits).  With z the argument of the logistic function and
    t = exp(-|z|) <= 1: the exponential is off by two units (4 x 2^-24 of its value), 1 + t, g t and the product with up by half a
    unit each, the quotient by two units; 11 x 2^-24 in all.  z itself is g (SiLU), or off by seven roundings of its terms, all of one
    sign (tanh-GELU), and moves the value by its error times one minus the logistic function, 1 / (1 + t) of it below zero and
    t / (1 + t) above.  Below 2^-126 t is off by 2^-148 and g t by another 2^-149."""
    if name == "silu":
        z, dz = g, 0.0
    else:
        z = 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
        dz = 7 * 2.0 ** -24 * np.abs(z)
    t = np.exp(-np.abs(z))
    value = np.where(z >= 0, g, g * t) / (1 + t)
    return value, (11 * 2.0 ** -24 + dz * np.where(z >= 0, t, 1.0) / (1 + t)) * np.abs(value) + 2.0 ** -148 * (np.abs(g) + 1)


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("y_dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,R,C,gate_byte,up_byte", [(1, 300, 2048, 124, 127), (40, 200, 64, 126, 127), (40, 64, 64, 121, 140), (300, 700, 96, 126, 126),
                                                     (40, 200, 64, 127, 150), (9, 333, 32, 190, 127), (300, 264, 32, 190, 127)])
def test_gates_far_from_zero(activation, y_dtype, n, R, C, gate_byte, up_byte):
    """Gates of up to a few hundred, and of up to 10^20, whose cube is infinite in 32 bits."""
    import torch
    if y_dtype == "f16" and (up_byte > 140 or gate_byte > 140):
        up_byte, gate_byte = min(up_byte, 134), min(gate_byte, 128)      # results that f16 holds
    handle, codes, bytes_ = pair(R + C, R, C, activation, gate_byte, up_byte)
    xc, xs, xv = rows(n, n, C)
    y = torch.full((n, R), 55.0, dtype=tt(y_dtype), device="cuda")
    torch.cuda.synchronize()
    assert handle.matmul(xc.data_ptr(), xs.data_ptr(), n, y.data_ptr(), y_dtype=y_dtype) == 0
    torch.cuda.synchronize()
    assert handle.status() == 0
    g, u = (xv @ eo.mx_values(c[0], b[0]).T for c, b in zip(codes, bytes_))
    with np.errstate(over="ignore"):
        a, err = act_in_steps(activation, g)
    want, err = a * u, err * np.abs(u)
    if y_dtype == "f16":
        inside = np.abs(want) + err < 65000
        assert inside.any()
        got = np.where(inside, y.double().cpu().numpy(), 0.0)
        eo.close(got, np.where(inside, want, 0.0), np.where(inside, err, 0.0), y_dtype)
    else:
        eo.close(y.double().cpu().numpy(), want, err, y_dtype)


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_pairs_that_are_not_numbers(activation, n):
    """A NaN block of the gate's row, of the up row or of an activation row makes the results that use it NaN, and no others."""
    import torch
    R, C = 150, 320
    rng = np.random.default_rng(n)
    code = [rng.integers(0, 16, (1, R, C)).astype(np.uint8) for _ in range(2)]
    byte = [np.full((1, R, C // 32), 124, np.uint8) for _ in range(2)]
    byte[0][0, 17, 3] = 255
    byte[1][0, 140, 9] = 255
    dev = [device(a) for c, b in zip(code, byte) for a in (eo.mx_pack(c), b)]
    handle = ex.Mxfp4Weights(R, C, 1, dev[0].data_ptr(), dev[1].data_ptr(), up_codes=dev[2].data_ptr(), up_scales=dev[3].data_ptr(),
                             activation=activation)
    xc, xs, _ = rows(n, n, C)
    xs[n // 2, 4] = 255
    y = torch.zeros(n, R, device="cuda")
    torch.cuda.synchronize()
    assert handle.matmul(xc.data_ptr(), xs.data_ptr(), n, y.data_ptr()) == 0
    torch.cuda.synchronize()
    want = np.zeros((n, R), bool)
    want[:, [17, 140]] = True
    want[n // 2] = True
    assert handle.status() == 0 and np.array_equal(torch.isnan(y).cpu().numpy(), want)
