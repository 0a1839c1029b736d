"""MXFP4 quantisation (codes and scales equal, bit for bit) and products (within the rounding of 32-bit sums) against the statement
in 64 bits."""
import importlib

import numpy as np
import pytest

import expert_ops_oracle as eo

pytestmark = pytest.mark.gpu
ex = importlib.import_module("salt-core_b200.experts")
TYPES = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def tt(name):
    import torch
    return getattr(torch, TYPES[name])


def quantize(x, dtype, index=None, div=1, rows=None, values=True, pad=0):
    """x: torch [n][cols] -> (codes packed, scales, values), the rows and bytes that are not written left at 0x5a."""
    import torch
    n, cols = x.shape
    held = torch.zeros(n, cols + pad, dtype=x.dtype, device="cuda")
    held[:, :cols] = x
    rows = n if rows is None else rows
    codes = torch.full((rows + 2, cols // 2), 0x5a, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows + 2, eo.scale_pitch(cols)), 0x5a, dtype=torch.uint8, device="cuda")
    vals = torch.full((rows + 2, cols), 55.0, dtype=x.dtype, device="cuda")
    torch.cuda.synchronize()
    assert ex.quantize(held.data_ptr(), n, cols, codes.data_ptr(), scales.data_ptr(), dtype=dtype, row_stride=cols + pad, rows=rows,
                       d_row_index=0 if index is None else index.data_ptr(), index_div=div,
                       d_values=vals.data_ptr() if values else 0) == 0
    torch.cuda.synchronize()
    return codes, scales, vals


def check_quantize(x, dtype, **k):
    import torch
    codes, scales, vals = quantize(x, dtype, **k)
    n, cols = x.shape
    code, byte = eo.mx_quantize(x.double().cpu().numpy())
    nb = cols // 32
    assert np.array_equal(scales[:n, :nb].cpu().numpy(), byte)
    assert np.array_equal(codes[:n].cpu().numpy(), eo.mx_pack(code))
    assert (scales[:, nb:] == 0x5a).all() and (scales[n:] == 0x5a).all() and (codes[n:] == 0x5a).all()
    want = torch.from_numpy(eo.mx_values(code, byte)).to(x.dtype).cuda()
    assert torch.equal(torch.nan_to_num(vals[:n], nan=77.0), torch.nan_to_num(want, nan=77.0)) and (vals[n:] == 55.0).all()
    assert torch.equal(torch.isnan(vals[:n]), torch.isnan(want))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,cols,pad", [(1, 32, 0), (3, 64, 8), (17, 96, 0), (5, 1056, 16), (130, 2816, 0), (2, 5120, 0)])
def test_quantize(dtype, n, cols, pad):
    import torch
    g = torch.Generator(device="cuda").manual_seed(n + cols)
    x = torch.randn(n, cols, device="cuda", generator=g) * torch.exp2(6 * torch.randn(n, cols, device="cuda", generator=g).clamp(-2, 1.5))
    check_quantize(x.to(tt(dtype)), dtype, pad=pad)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantize_every_tie_and_extreme(dtype):
    """All halfway values at many scales, both signs; zeros; subnormals; the largest finite value; infinities and NaN."""
    import torch
    t = tt(dtype)
    info = torch.finfo(t)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.75, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0]).repeat(2)
    ties[16:] *= -1
    ties[15] = 4.0
    rows = [ties * 2.0 ** e for e in (range(-9, 13) if dtype == "f16" else range(-120, 125, 7))]
    zero = torch.zeros(32)
    zero[::2] = -0.0
    rows += [zero, torch.full((32,), info.max), torch.full((32,), info.tiny), torch.full((32,), info.smallest_normal / 4)]
    rows.append(torch.linspace(-1, 1, 32) * info.tiny)
    for bad in (torch.nan, torch.inf, -torch.inf):
        r = torch.ones(32)
        r[7] = bad
        rows.append(r)
    check_quantize(torch.stack(rows).to(t).cuda(), dtype)


def test_quantize_by_index():
    """Rows in grouped order, the same row several times; an index below zero or beyond the rows leaves its row alone."""
    import torch
    T, k, cols = 21, 4, 160
    x = torch.randn(T, cols, device="cuda").bfloat16()
    index = torch.randperm(T * k, device="cuda").to(torch.int32)
    index[[0, 9, 30]] = torch.tensor([-1, T * k, -2 ** 31], dtype=torch.int32, device="cuda")
    codes, scales, vals = quantize(x, "bf16", index, k, T * k)
    code, byte = eo.mx_quantize(x.double().cpu().numpy())
    for i, at in enumerate(index.tolist()):
        if 0 <= at < T * k:
            assert np.array_equal(codes[i].cpu().numpy(), eo.mx_pack(code[at // k])), i
            assert np.array_equal(scales[i, :5].cpu().numpy(), byte[at // k]), i
        else:
            assert (codes[i] == 0x5a).all() and (scales[i] == 0x5a).all() and (vals[i] == 55.0).all()
    assert (codes[T * k:] == 0x5a).all()
    again = quantize(x, "bf16", index, k, T * k, values=False)
    assert torch.equal(again[0], codes) and torch.equal(again[1], scales) and (again[2] == 55.0).all()


def weights(rng, *shape):
    """Random matrices as codes and scale bytes [..., rows, cols], every code among them, scales over a few binades."""
    code = rng.integers(0, 16, shape).astype(np.uint8)
    byte = rng.integers(118, 127, (*shape[:-1], shape[-1] // 32)).astype(np.uint8)
    return code, byte


def device(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Held:
    """A handle and the values its matrices stand for."""

    def __init__(self, seed, E, R, C, activation=None, host=False):
        rng = np.random.default_rng(seed)
        self.parts = [weights(rng, E, R, C) for _ in range(2 if activation else 1)]
        packed = [(eo.mx_pack(c), b) for c, b in self.parts]
        if not host:
            packed = [(device(c), device(b)) for c, b in packed]
        addr = [a.ctypes.data if host else a.data_ptr() for p in packed for a in p]
        self.activation = activation
        self.handle = ex.Mxfp4Weights(R, C, E, *addr[:2], **(dict(up_codes=addr[2], up_scales=addr[3], activation=activation)
                                                             if activation else {}))
        self.values = [eo.mx_values(c, b) for c, b in self.parts]

    def want(self, xv, e=0):
        if self.activation:
            return eo.gated(self.activation, xv, self.values[0][e], self.values[1][e])
        return eo.product(xv, self.values[0][e])


def acts(seed, n, C, dtype="f32"):
    """Quantised rows on the device and the values they stand for."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(max(n, 1), C, device="cuda", generator=g).to(tt(dtype))[:n]
    codes, scales, _ = quantize(x, dtype)
    code, byte = eo.mx_quantize(x.double().cpu().numpy()) if n else (np.zeros((0, C), np.uint8), np.zeros((0, C // 32), np.uint8))
    return codes, scales, eo.mx_values(code, byte)


def check_matmul(held, n, R, C, y_dtype="f32", y_pad=0, seed=0):
    import torch
    codes, scales, xv = acts(seed + n, n, C)
    y = torch.full((n + 1, R + y_pad), 55.0, dtype=tt(y_dtype), device="cuda")
    torch.cuda.synchronize()
    assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr(), y_dtype=y_dtype, y_row_stride=R + y_pad) == 0
    torch.cuda.synchronize()
    assert held.handle.status() == 0
    want, err = held.want(xv)
    eo.close(y[:n, :R].double().cpu().numpy(), want, err, y_dtype, f"{n} rows of {R} x {C}")
    assert (y[n:] == 55.0).all() and (y[:, R:] == 55.0).all()


SHAPES = [(1, 32), (7, 64), (64, 96), (129, 288), (128, 256), (300, 1056), (704, 2816), (257, 544)]


@pytest.mark.parametrize("R,C", SHAPES)
@pytest.mark.parametrize("activation", [None, "silu", "gelu_tanh"])
def test_matmul_shapes(R, C, activation):
    held = Held(R + C, 1, R, C, activation)
    for n in (1, 2, 3, 5, 8, 9, 16, 17, 33, 64, 65, 129, 300):
        check_matmul(held, n, R, C, seed=R)


@pytest.mark.parametrize("y_dtype", list(TYPES))
@pytest.mark.parametrize("y_pad", [0, 1, 8])
@pytest.mark.parametrize("activation", [None, "silu"])
def test_matmul_results(y_dtype, y_pad, activation):
    held = Held(11, 1, 203, 320, activation, host=True)
    for n in (1, 4, 50, 140):
        check_matmul(held, n, 203, 320, y_dtype, y_pad)


@pytest.mark.parametrize("n,R,C,activation", [(500, 1300, 1056, None), (1000, 700, 544, "silu"), (230, 20000, 288, None), (4099, 300, 96, None),
                                              (449, 129, 800, "gelu_tanh"), (97, 5000, 512, None), (225, 2050, 2080, "silu")])
@pytest.mark.parametrize("y_dtype", ["f32", "bf16"])
def test_matmul_many_rows(n, R, C, activation, y_dtype):
    """Passes of more than 96 rows, an odd number of row tiles among them, more units than places on the chip."""
    check_matmul(Held(n, 1, R, C, activation), n, R, C, y_dtype, seed=R)


def test_wide_rows():
    """Rows at the documented limit, and one that leaves room for fewer tokens a pass."""
    for C in (131072, 40960):
        held = Held(C, 1, 40, C)
        for n in (1, 6, 20):
            check_matmul(held, n, 40, C)


def test_no_rows():
    held = Held(3, 2, 32, 64)
    assert held.handle.experts(0, 0, 0x1000, 0, 0) == 0
    assert Held(3, 1, 32, 64).handle.matmul(0, 0, 0, 0) == 0


def test_bad_scales_stay_where_they_are():
    """A NaN block of an activation row or of a weight row makes the results that use it NaN, and no others."""
    import torch
    R, C = 70, 512
    rng = np.random.default_rng(8)
    code, byte = weights(rng, 1, R, C)
    byte[0, 13, 5] = 255
    w = [device(eo.mx_pack(code)), device(byte)]
    handle = ex.Mxfp4Weights(R, C, 1, w[0].data_ptr(), w[1].data_ptr())
    for n in (1, 3, 8, 40, 130):
        x = torch.randn(n, C, device="cuda")
        x[n // 2, 100] = torch.nan
        codes, scales, _ = quantize(x, "f32")
        y = torch.empty(n, R, device="cuda")
        assert handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr()) == 0
        nan = torch.isnan(y).cpu().numpy()
        want = np.zeros((n, R), bool)
        want[:, 13] = True
        want[n // 2] = True
        assert np.array_equal(nan, want), n


GROUPS = {"token": [1, 0, 1, 0, 0, 1], "even": [3, 3, 3, 3, 3, 3], "one": [0, 0, 40, 0, 0, 0], "ragged": [1, 17, 0, 130, 5, 64],
          "last": [0, 0, 0, 0, 0, 9], "large": [240, 1, 300, 225, 16, 224]}


@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("R,C,activation", [(96, 288, "silu"), (200, 512, None), (64, 96, "gelu_tanh"), (129, 1056, None)])
def test_experts(name, R, C, activation):
    """Groups of every size, empty ones, rows behind the last group, whose outputs stay."""
    import torch
    counts = GROUPS[name]
    E, live, behind = len(counts), sum(counts), 5
    held = Held(R + live, E, R, C, activation)
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    n = live + behind
    codes, scales, xv = acts(live, n, C, "bf16")
    off = device(offsets)
    y = torch.full((n, R), 55.0, device="cuda")
    torch.cuda.synchronize()
    assert held.handle.experts(codes.data_ptr(), scales.data_ptr(), off.data_ptr(), n, y.data_ptr()) == 0
    torch.cuda.synchronize()
    assert held.handle.status() == 0
    got = y.double().cpu().numpy()
    for e in range(E):
        b, t = offsets[e], offsets[e + 1]
        if t > b:
            want, err = held.want(xv[b:t], e)
            eo.close(got[b:t], want, err, "f32", f"expert {e}")
    assert (got[live:] == 55.0).all()


@pytest.mark.parametrize("R,C,activation", [(1300, 800, None), (650, 544, "silu"), (64, 2080, "gelu_tanh")])
def test_experts_of_long_groups(R, C, activation):
    """Groups around the largest pass, and a popular expert with several."""
    import torch
    counts = [224, 0, 225, 97, 700, 1, 448]
    E, live = len(counts), sum(counts)
    held = Held(R, E, R, C, activation)
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    codes, scales, xv = acts(3, live, C)
    off, y = device(offsets), torch.full((live, R), 55.0, device="cuda")
    torch.cuda.synchronize()
    assert held.handle.experts(codes.data_ptr(), scales.data_ptr(), off.data_ptr(), live, y.data_ptr()) == 0
    torch.cuda.synchronize()
    assert held.handle.status() == 0
    got = y.double().cpu().numpy()
    for e in range(E):
        b, t = offsets[e], offsets[e + 1]
        if t > b:
            want, err = held.want(xv[b:t], e)
            eo.close(got[b:t], want, err, "f32", f"expert {e}")


def test_many_experts():
    """1024 experts, most of them empty."""
    import torch
    E, R, C = 1024, 32, 64
    held = Held(77, E, R, C)
    counts = np.zeros(E, np.int64)
    counts[[0, 5, 500, 1022, 1023]] = [2, 1, 30, 3, 9]
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    n = int(counts.sum())
    codes, scales, xv = acts(4, n, C)
    off, y = device(offsets), torch.zeros(n, R, device="cuda")
    torch.cuda.synchronize()
    assert held.handle.experts(codes.data_ptr(), scales.data_ptr(), off.data_ptr(), n, y.data_ptr()) == 0
    got = y.double().cpu().numpy()
    for e in np.nonzero(counts)[0]:
        want, err = held.want(xv[offsets[e]:offsets[e + 1]], e)
        eo.close(got[offsets[e]:offsets[e + 1]], want, err, "f32", f"expert {e}")


def test_strided_weights():
    """Experts laid out as slots of gate codes | gate scales | up codes | up scales, scale rows further apart than they are long."""
    import torch
    E, R, C, pitch = 3, 40, 96, 7
    rng = np.random.default_rng(2)
    parts = [weights(rng, E, R, C) for _ in range(2)]
    slot = 2 * (R * C // 2 + R * pitch) + 13
    pool = np.zeros((E, slot), np.uint8)
    for e in range(E):
        at = 0
        for code, byte in parts:
            pool[e, at:at + R * C // 2] = eo.mx_pack(code[e]).reshape(-1)
            at += R * C // 2
            rows = np.full((R, pitch), 0xff, np.uint8)
            rows[:, :C // 32] = byte[e]
            pool[e, at:at + R * pitch] = rows.reshape(-1)
            at += R * pitch
    d, half = device(pool), R * C // 2 + R * pitch
    base = d.data_ptr()
    handle = ex.Mxfp4Weights(R, C, E, base, base + R * C // 2, up_codes=base + half, up_scales=base + half + R * C // 2, activation="silu",
                             expert_code_stride=slot, expert_scale_stride=slot, scale_row_stride=pitch)
    off = device(np.array([0, 2, 5, 6], np.int32))
    codes, scales, xv = acts(1, 6, C)
    y = torch.zeros(6, R, device="cuda")
    torch.cuda.synchronize()
    assert handle.experts(codes.data_ptr(), scales.data_ptr(), off.data_ptr(), 6, y.data_ptr()) == 0
    got = y.double().cpu().numpy()
    for e, (b, t) in enumerate(((0, 2), (2, 5), (5, 6))):
        want, err = eo.gated("silu", xv[b:t], *[eo.mx_values(c[e], s[e]) for c, s in parts])
        eo.close(got[b:t], want, err, "f32")


def test_refusals_with_a_handle():
    held = Held(1, 2, 32, 64)
    h, P = held.handle, 0x1000
    assert h.matmul(P, P, 1, P) == -1                    # two experts: not one matrix
    assert h.experts(P, P, 0, 1, P) == -1
    for bad in (dict(d_codes=0), dict(d_scales=0), dict(d_y=0), dict(rows=-1), dict(d_codes=P + 8), dict(d_scales=P + 1), dict(d_y=P + 2),
                dict(y_row_stride=31)):
        assert h.experts(**{**dict(d_codes=P, d_scales=P, d_group_offsets=P, rows=1, d_y=P), **bad}) == -1, bad
    assert h.lib.salt_b200_mxfp4_experts(h.handle, P, P, P, 1, P, 3, 32, 0) == -1


@pytest.mark.parametrize("n", [1, 7, 90, 400])
def test_repeated_and_captured(n):
    """The same bits again, on another stream, and replayed from a graph on new activations."""
    import torch
    R, C = 300, 1056
    held = Held(6, 1, R, C)
    codes, scales, xv = acts(5, n, C)
    y, z = torch.empty(n, R, device="cuda"), torch.empty(n, R, device="cuda")
    torch.cuda.synchronize()
    assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr()) == 0
    s = torch.cuda.Stream()
    assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, z.data_ptr(), stream=s.cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(y, z)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, z.data_ptr(), stream=torch.cuda.current_stream().cuda_stream) == 0
    new = acts(6, n, C)
    codes.copy_(new[0])
    scales.copy_(new[1])
    g.replay()
    torch.cuda.synchronize()
    want, err = held.want(new[2])
    eo.close(z.double().cpu().numpy(), want, err, "f32")


@pytest.mark.parametrize("n", [1, 40, 130, 400])
def test_scales_far_from_one(n):
    """Weights of 2^-107 with activations of 2^103 and the other way round: their products are near one."""
    import torch
    R, C = 300, 512
    rng = np.random.default_rng(n)
    for wb, xe in ((20, 100), (225, -104)):
        code = rng.integers(0, 16, (1, R, C)).astype(np.uint8)
        byte = rng.integers(wb - 2, wb + 3, (1, R, C // 32)).astype(np.uint8)
        dev = [device(eo.mx_pack(code)), device(byte)]
        handle = ex.Mxfp4Weights(R, C, 1, dev[0].data_ptr(), dev[1].data_ptr())
        x = torch.randn(n, C, device="cuda") * 2.0 ** xe
        codes, scales, _ = quantize(x, "f32")
        xv = eo.mx_values(*eo.mx_quantize(x.double().cpu().numpy()))
        y = torch.empty(n, R, device="cuda")
        assert handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr()) == 0
        want, err = eo.product(xv, eo.mx_values(code, byte)[0])
        eo.close(y.double().cpu().numpy(), want, err, "f32", f"scales of {wb}")


@pytest.mark.parametrize("R,activation", [(96, None), (700, "silu")])
def test_groups_that_end_early_or_late(R, activation):
    """No group has a row: nothing is written.  Offsets behind `rows`: rows up to there are computed, the others stay."""
    import torch
    E, C, n = 5, 544, 130
    held = Held(R, E, R, C, activation)
    codes, scales, xv = acts(9, n, C)
    y = torch.full((n, R), 55.0, device="cuda")
    none = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    for rows in (1, n):
        assert held.handle.experts(codes.data_ptr(), scales.data_ptr(), none.data_ptr(), rows, y.data_ptr()) == 0
    torch.cuda.synchronize()
    assert held.handle.status() == 0 and (y == 55.0).all()
    off = device(np.array([0, 3, 50, 120, 125, 300], np.int32))
    rows = 119
    assert held.handle.experts(codes.data_ptr(), scales.data_ptr(), off.data_ptr(), rows, y.data_ptr()) == 0
    torch.cuda.synchronize()
    assert held.handle.status() == 0 and (y[rows:] == 55.0).all()
    got = y.double().cpu().numpy()
    for e, (b, t) in enumerate(((0, 3), (3, 50), (50, 119))):
        want, err = held.want(xv[b:t], e)
        eo.close(got[b:t], want, err, "f32", f"expert {e}")


def test_two_streams_at_once():
    """One handle used on two streams at the same time, calls of every launch form side by side."""
    import torch
    R, C = 1300, 1056
    held = Held(21, 1, R, C)
    sizes = (1, 300, 8, 90, 700, 2)
    data = [acts(n, n, C) for n in sizes]
    ys = [[torch.empty(n, R, device="cuda") for n in sizes] for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for turn in range(6):
        for k, s in enumerate(streams):
            for i in (range(len(sizes)) if k == 0 else reversed(range(len(sizes)))):
                assert held.handle.matmul(data[i][0].data_ptr(), data[i][1].data_ptr(), sizes[i], ys[k][i].data_ptr(), stream=s.cuda_stream) == 0
    torch.cuda.synchronize()
    assert held.handle.status() == 0
    for i in range(len(sizes)):
        assert torch.equal(ys[0][i], ys[1][i])
        want, err = held.want(data[i][2])
        eo.close(ys[0][i].double().cpu().numpy(), want, err, "f32", f"{sizes[i]} rows")


def test_quantize_and_product_back_to_back():
    """The same buffers quantised and multiplied again and again: a launch that starts early does not touch what the one before reads."""
    import torch
    n, R, C = 37, 700, 2080
    held = Held(31, 1, R, C)
    xs = [torch.randn(n, C, device="cuda") for _ in range(12)]
    codes = torch.empty(n, C // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n, eo.scale_pitch(C), dtype=torch.uint8, device="cuda")
    ys = [torch.empty(n, R, device="cuda") for _ in xs]
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        assert ex.quantize(x.data_ptr(), n, C, codes.data_ptr(), scales.data_ptr()) == 0
        assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr()) == 0
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        want, err = held.want(eo.mx_values(*eo.mx_quantize(x.double().cpu().numpy())))
        eo.close(y.double().cpu().numpy(), want, err, "f32")


def test_rows_beyond_32_bits():
    """Row numbers whose byte offsets in codes and results pass 2^32: 2.2 million rows of 4096 columns, all of them zeros but a few."""
    import torch
    n, R, C = 2_200_003, 520, 4096
    held = Held(41, 1, R, C)
    codes = torch.zeros(n, C // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, eo.scale_pitch(C)), 127, dtype=torch.uint8, device="cuda")
    at = [0, 1_048_577, 2_097_160, n - 1]
    few = acts(3, len(at), C)
    codes[at], scales[at] = few[0][:len(at)], few[1][:len(at)]
    y = torch.full((n, R), 55.0, device="cuda")
    torch.cuda.synchronize()
    assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr()) == 0
    torch.cuda.synchronize()
    assert held.handle.status() == 0
    want, err = held.want(few[2])
    eo.close(y[at].double().cpu().numpy(), want, err, "f32")
    y[at] = 0
    assert not y.any()


def coded(seed, n, C):
    """Random codes and scales as activations, and the values they stand for."""
    rng = np.random.default_rng(seed)
    code, byte = weights(rng, n, C)
    held = np.full((n, eo.scale_pitch(C)), 0xff, np.uint8)               # the bytes behind the blocks are not read
    held[:, :C // 32] = byte
    return device(eo.mx_pack(code)), device(held), eo.mx_values(code, byte)


# (rows, R, C, activation, groups or None, runs on pairs of SMs): shapes that reach the launch forms of long passes
LONG = [(770, 1300, 5056, None, None, True), (800, 700, 5024, "silu", None, False), (2000, 1030, 5024, "silu", None, True),
        (1537, 1409, 4000, "gelu_tanh", None, True), (1001, 2817, 2848, None, None, True),
        (1500, 130, 7968, "gelu_tanh", None, False), (3000, 5000, 1056, None, None, False),
        (97, 1, 8032, None, None, False), (300, 100, 8032, None, None, False), (150, 60, 5440, "silu", None, False),
        (18889, 64, 1408, None, None, False), (20000, 100, 1440, None, None, False), (19000, 50, 1408, "silu", None, False),
        (2600, 1300, 1568, None, [700, 0, 224, 225, 226, 900, 1, 324], True), (2600, 650, 1568, "silu", [0, 2600, 0, 0, 0, 0, 0, 0], True),
        (14967, 64, 1376, None, [7000, 0, 7967], False)]


@pytest.mark.parametrize("n,R,C,activation,groups,pair", LONG)
@pytest.mark.parametrize("y_dtype,y_pad", [("bf16", 0), ("f32", 3), ("f16", 8)])
def test_long_passes(n, R, C, activation, groups, pair, y_dtype, y_pad):
    import torch
    from graph_util import captured_kernels
    counts = groups or [n]
    E = len(counts)
    held = Held(R + C, E, R, C, activation)
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    codes, scales, xv = coded(n, n, C)
    off, y = device(offsets), torch.full((n + 1, R + y_pad), 55.0, dtype=tt(y_dtype), device="cuda")
    torch.cuda.synchronize()

    def call(stream=0):
        if groups:
            rc = held.handle.experts(codes.data_ptr(), scales.data_ptr(), off.data_ptr(), n, y.data_ptr(), y_dtype=y_dtype, y_row_stride=R + y_pad,
                                     stream=stream)
        else:
            rc = held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr(), y_dtype=y_dtype, y_row_stride=R + y_pad, stream=stream)
        assert rc == 0
    call()
    torch.cuda.synchronize()
    assert held.handle.status() == 0
    got = y.double().cpu().numpy()
    assert (got[n:] == 55.0).all() and (got[:, R:] == 55.0).all()
    for e in range(E):
        b, t = offsets[e], offsets[e + 1]
        if t > b:
            want, err = held.want(xv[b:t], e)
            eo.close(got[b:t, :R], want, err, y_dtype, f"group {e}")
    (name, grid), = captured_kernels(call)
    assert ("ELb1EEEv" in name) == pair, (name, grid)


def test_pairs_repeat_their_bits():
    """Long passes, twice in a row, on a busy chip and captured: the same bits."""
    import torch
    n, R, C = 1001, 2817, 2848
    held = Held(5, 1, R, C)
    codes, scales, _ = coded(1, n, C)
    ys = [torch.empty(n, R, device="cuda") for _ in range(6)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i, y in enumerate(ys[:5]):
        assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, y.data_ptr(), stream=streams[i % 2].cuda_stream) == 0
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert held.handle.matmul(codes.data_ptr(), scales.data_ptr(), n, ys[5].data_ptr(), stream=torch.cuda.current_stream().cuda_stream) == 0
    g.replay()
    torch.cuda.synchronize()
    assert held.handle.status() == 0
    for y in ys[1:]:
        assert torch.equal(y, ys[0])


@pytest.mark.parametrize("activation", [None, "silu"])
def test_host_weights_of_several_experts_and_a_single_group(activation):
    """Weights from host memory, gone after the handle is made; and a handle of one expert called by groups."""
    import gc
    import torch
    for E, counts in ((3, [2, 0, 70]), (1, [45])):
        held = Held(60 + E, E, 140, 544, activation, host=True)
        gc.collect()
        offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        n = int(offsets[-1])
        codes, scales, xv = acts(n, n, 544, "f16")
        off, y = device(offsets), torch.empty(n, 140, device="cuda")
        torch.cuda.synchronize()
        assert held.handle.experts(codes.data_ptr(), scales.data_ptr(), off.data_ptr(), n, y.data_ptr()) == 0
        got = y.double().cpu().numpy()
        for e in range(E):
            b, t = offsets[e], offsets[e + 1]
            if t > b:
                want, err = held.want(xv[b:t], e)
                eo.close(got[b:t], want, err, "f32", f"expert {e} of {E}")


def test_weights_of_quantized_rows():
    """Weights quantised on the device, their scale rows as the quantiser leaves them, straight into a handle."""
    import torch
    R, C, n = 300, 1056, 19
    w = torch.randn(R, C, device="cuda").bfloat16() / 32
    codes, scales, _ = quantize(w, "bf16")
    handle = ex.Mxfp4Weights(R, C, 1, codes.data_ptr(), scales.data_ptr(), scale_row_stride=eo.scale_pitch(C))
    xc, xs, xv = acts(2, n, C, "bf16")
    y = torch.empty(n, R, device="cuda")
    assert handle.matmul(xc.data_ptr(), xs.data_ptr(), n, y.data_ptr()) == 0
    want, err = eo.product(xv, eo.mx_values(*eo.mx_quantize(w.double().cpu().numpy())))
    eo.close(y.double().cpu().numpy(), want, err, "f32")
