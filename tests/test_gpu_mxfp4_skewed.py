"""Expert products of a layer's width whose tokens are far from evenly shared, as routers leave them: the pass size follows the average
group, so some groups need many passes and others a part of one."""
import importlib

import numpy as np
import pytest

import expert_ops_oracle as eo

pytestmark = pytest.mark.gpu
ex = importlib.import_module("salt-core_b200.experts")


def shares(name, E, n):
    """Rows of every expert, n in all."""
    rng = np.random.default_rng(E + n)
    if name == "one":                                    # three quarters to one expert, single rows to a few others
        c = np.zeros(E, np.int64)
        c[rng.choice(E, E // 4, replace=False)] = 1
    else:
        p = 1.0 / np.arange(1, E + 1) ** (1.0 if name == "harmonic" else 2.0)
        c = np.floor(n * rng.permutation(p / p.sum())).astype(np.int64)
    c[np.argmax(c)] += n - c.sum()
    return c


def dequantised(codes, scales):
    import torch
    grid = torch.tensor(np.concatenate((eo.GRID, -eo.GRID)), device="cuda")
    both = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    return grid[both.long()] * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


@pytest.mark.parametrize("name", ["one", "harmonic", "square"])
@pytest.mark.parametrize("E,R,C,activation,n,y_dtype", [(64, 1536, 2560, "silu", 4003, "bf16"), (128, 704, 2816, "gelu_tanh", 511, "f32"),
                                                        (64, 2560, 1536, None, 4003, "bf16"), (31, 700, 1056, "silu", 9001, "f16")])
def test_skewed_groups(name, E, R, C, activation, n, y_dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(n + E)
    first, behind = 5, 3                                 # rows before the first group and behind the last

    def some(low, high, *shape):
        return torch.randint(low, high, shape, dtype=torch.uint8, device="cuda", generator=g)
    parts = [(some(0, 256, E, R, C // 2), some(118, 124, E, R, C // 32)) for _ in range(2 if activation else 1)]
    handle = ex.Mxfp4Weights(R, C, E, *[t.data_ptr() for t in parts[0]], activation=activation,
                             **(dict(up_codes=parts[1][0].data_ptr(), up_scales=parts[1][1].data_ptr()) if activation else {}))
    rows = first + n + behind
    xc, xs = some(0, 256, rows, C // 2), some(118, 124, rows, ex.scale_pitch(C))
    offsets = first + np.concatenate(([0], np.cumsum(shares(name, E, n))))
    off = torch.from_numpy(offsets.astype(np.int32)).cuda()
    y = torch.full((rows, R), 55.0, dtype={"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[y_dtype], device="cuda")
    torch.cuda.synchronize()
    assert handle.experts(xc.data_ptr(), xs.data_ptr(), off.data_ptr(), rows, y.data_ptr(), y_dtype=y_dtype) == 0
    torch.cuda.synchronize()
    assert handle.status() == 0
    assert (y[:first] == 55.0).all() and (y[first + n:] == 55.0).all()
    x, got = dequantised(xc, xs[:, :C // 32]), y.double().cpu().numpy()
    for e in range(E):
        b, t = offsets[e], offsets[e + 1]
        if t == b:
            continue
        # products and the sums of their magnitudes as in expert_ops_oracle.product, on the device
        sums = []
        for codes, scales in parts:
            w = dequantised(codes[e], scales[e])
            sums.append(((x[b:t] @ w.T).cpu().numpy(), (C / 32 + 8) * 2.0 ** -23 * (x[b:t].abs() @ w.abs().T).cpu().numpy()))
        want, err = sums[0]
        if activation:
            (gate, eg), (up, eu) = sums
            a = eo.act(activation, gate)
            want, err = a * up, (1.13 * eg + 2.0 ** -21 * np.abs(gate)) * (np.abs(up) + eu) + np.abs(a) * eu
        eo.close(got[b:t], want, err, y_dtype, f"expert {e}")
