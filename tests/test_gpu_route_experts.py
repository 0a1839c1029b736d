"""Routing and grouping outside a stack against the statement in 64 bits: selections and groupings are whole numbers and equal,
weights are within the rounding of 32 bits."""
import importlib

import numpy as np
import pytest

import expert_ops_oracle as eo

pytestmark = pytest.mark.gpu
ex = importlib.import_module("salt-core_b200.experts")
TYPES = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def run(logits, topk, dtype="f32", bias=None, group=True, pad=0, stream=0, **k):
    """logits: a torch tensor on the device; pad: columns behind every row."""
    import torch
    T, E = logits.shape
    held = torch.full((T, E + pad), 99.0, dtype=logits.dtype, device="cuda")
    held[:, :E] = logits
    n = T * topk
    sel = torch.full((n + 8,), 77, dtype=torch.int32, device="cuda")
    w = torch.full((n + 8,), 77.0, device="cuda")
    off, g2c, c2g = (torch.full((m + 8,), 77, dtype=torch.int32, device="cuda") for m in (E + 1, n, n))
    b = None if bias is None else torch.as_tensor(np.asarray(bias, np.float32)).cuda()
    torch.cuda.synchronize()
    rc = ex.route(ex.RouteSpec(E, topk, **k), held.data_ptr(), T, sel.data_ptr(), w.data_ptr(),
                  *([t.data_ptr() for t in (off, g2c, c2g)] if group else []), dtype=dtype, row_stride=E + pad,
                  d_bias=0 if b is None else b.data_ptr(), stream=stream)
    assert rc == 0
    torch.cuda.synchronize()
    for t, m in ((sel, n), (w, n), (off, E + 1 if group else 0), (g2c, n if group else 0), (c2g, n if group else 0)):
        assert (t[m:] == 77).all()                       # nothing behind the results is touched
    return (sel[:n].view(T, topk).cpu().numpy(), w[:n].view(T, topk).cpu().numpy(), off[:E + 1].cpu().numpy(), g2c[:n].cpu().numpy(),
            c2g[:n].cpu().numpy())


def check(logits, topk, dtype="f32", bias=None, group=True, pad=0, **k):
    T, E = logits.shape
    sel, w, off, g2c, c2g = run(logits, topk, dtype, bias, group, pad, **k)
    want, ww = eo.route(logits.double().cpu().numpy(), topk, bias=None if bias is None else np.asarray(bias, np.float32), **k)
    assert np.array_equal(sel, want)
    # a score: exponential 2 units, difference |l - m| / 2 units (below 60 here), sum 40, division, weight and scale 3: 2^-24 each
    eo.close(w, ww, 110 * 2.0 ** -24 * np.abs(ww), "f32", "weights")
    if group:
        for a, b, name in zip((off, g2c, c2g), eo.grouping(want, E), ("offsets", "g2c", "c2g")):
            assert np.array_equal(a, b), name


def logits_of(seed, T, E, dtype, spread=2.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (spread * torch.randn(T, E, device="cuda", generator=g)).to(getattr(torch, TYPES[dtype]))


@pytest.mark.parametrize("T", [1, 2, 16, 17, 255, 700])
@pytest.mark.parametrize("E,topk", [(1, 1), (8, 2), (31, 5), (64, 4), (128, 8), (257, 8), (1024, 32)])
def test_softmax(T, E, topk):
    if T * E > 300000:
        T = 290
    check(logits_of(E + T, T, E, "f32"), topk, renormalize=T % 2 == 0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,G,keep,top", [(256, 8, 4, 2), (60, 4, 2, 1), (96, 32, 5, 2), (21, 3, 2, 2), (512, 16, 16, 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_groups(dtype, scoring, E, G, keep, top, biased):
    bias = 0.2 * np.random.default_rng(E).standard_normal(E) if biased else None
    check(logits_of(E, 67, E, dtype), 4, dtype, bias, scoring=scoring, n_groups=G, topk_groups=keep, group_top=top, pad=3, scale=2.5)


def test_keys_closer_than_32_bits():
    """Two experts whose keys differ by less than a rounding of the scores: the order is that of 64 bits."""
    import torch
    rng = np.random.default_rng(5)
    T, E = 64, 128
    l = rng.standard_normal((T, E)).astype(np.float32)
    bias = np.zeros(E, np.float32)
    # sigmoid near 1/2 is 1/2 + l / 4: the two differ by 2^-29 and the smaller index is not always the larger key
    for t in range(T):
        a, b = rng.choice(E, 2, replace=False)
        l[t] = -3.0
        l[t, a], l[t, b] = 2.0 ** -9, 2.0 ** -9 + 2.0 ** -27
    for k in (dict(), dict(n_groups=4, topk_groups=1, group_top=1), dict(n_groups=8, topk_groups=2, group_top=2)):
        check(torch.from_numpy(l).cuda(), 1, bias=bias, scoring="sigmoid", **k)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_equal_logits_and_masks(scoring, biased, groups):
    """Ties go to the lowest index; rows with few experts left, with none, with infinities, NaN and the lowest value."""
    import torch
    E = 32
    low = torch.finfo(torch.float32).min
    rows = torch.zeros(12, E)
    rows[1] = -torch.inf
    rows[2] = torch.nan
    rows[3, 3:] = -torch.inf
    rows[4, ::2] = torch.nan
    rows[5] = low
    rows[6] = low
    rows[6, 9] = 0.0
    rows[7, 4] = torch.inf
    rows[8, 20:24] = torch.inf
    rows[9] = -0.0
    rows[9, 5] = 0.0
    rows[10] = torch.arange(E) % 4
    rows[11, 1:] = -torch.inf
    bias = np.where(np.arange(E) % 8 == 7, -np.inf, 0.0) if biased else None
    for renorm in (True, False):
        check(rows.cuda(), 6, bias=bias, scoring=scoring, n_groups=groups, topk_groups=min(groups, 2), group_top=2, renormalize=renorm)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_bias_that_is_not_a_number(scoring, groups):
    """A bias of NaN or -infinity takes an expert out, +infinity puts it first; neither enters a weight."""
    bias = np.linspace(-0.2, 0.2, 64)
    bias[[3, 20]], bias[[7, 40]], bias[[12, 55]] = np.nan, -np.inf, np.inf
    check(logits_of(8, 70, 64, "f32"), 5, bias=bias, scoring=scoring, n_groups=groups, topk_groups=min(groups, 3), group_top=1)


def test_more_selections_than_registers_hold():
    """65536 selections and more: a warp's piece is longer than what it keeps between its two passes; all for one expert, too."""
    import torch
    for T, E, topk, spread in ((9001, 64, 8, 2.0), (70000, 16, 1, 2.0), (70000, 600, 1, 2.0), (70000, 8, 1, 0.0)):
        l = logits_of(T, T, E, "f32", spread)
        sel, w, off, g2c, c2g = run(l, topk)
        order = torch.sort(torch.from_numpy(sel.reshape(-1).astype(np.int64)), stable=True).indices.numpy()
        assert np.array_equal(g2c, order) and np.array_equal(c2g[g2c], np.arange(T * topk))
        assert np.array_equal(off, np.concatenate(([0], np.cumsum(np.bincount(sel.reshape(-1), minlength=E)))))
        want = torch.sort(l.double(), dim=1, descending=True, stable=True).indices[:, :topk].sort(dim=1).values
        assert np.array_equal(sel, want.cpu().numpy())


def test_scores_too_small_for_32_bits():
    import torch
    l = torch.full((3, 64), -300.0, device="cuda") - torch.arange(64, device="cuda")[None]
    l[1] -= 300.0
    l[2] -= 1e6                                          # and too small for 64: the weights are zeros
    sel, w, *_ = run(l, 4, scoring="sigmoid")
    want, ww = eo.route(l.double().cpu().numpy(), 4, scoring="sigmoid")
    assert np.array_equal(sel, want)
    eo.close(w, ww, 2.0 ** -22 * ww, "f32")
    assert not w[2].any() and w[0].sum() > 0.99


@pytest.mark.parametrize("T", [0, 1, 16, 17, 300, 4099])
@pytest.mark.parametrize("E,topk", [(4, 4), (128, 8), (1024, 3)])
def test_grouping(T, E, topk):
    """Groupings of every size, one expert that takes all of them among them."""
    import torch
    l = torch.zeros(max(T, 1), E, device="cuda") if T % 2 else logits_of(T + E, max(T, 1), E, "f32")
    l = l[:T]
    sel, w, off, g2c, c2g = run(l, topk)
    ref = torch.sort(torch.from_numpy(sel.reshape(-1).astype(np.int64)), stable=True).indices.numpy()
    assert np.array_equal(g2c, ref)
    assert np.array_equal(off, np.concatenate(([0], np.cumsum(np.bincount(sel.reshape(-1), minlength=E)))))
    assert np.array_equal(c2g[g2c], np.arange(T * topk))
    assert (np.diff(sel, axis=1) > 0).all()


def test_without_grouping_and_repeated():
    l = logits_of(3, 40, 128, "bf16")
    first = run(l, 8, "bf16", group=False)
    again = run(l, 8, "bf16")
    for a, b in zip(first[:2], again[:2]):
        assert a.tobytes() == b.tobytes()


def test_captured():
    """A routing captured into a graph, replayed on new logits; on a stream of its own."""
    import torch
    E, topk = 256, 8
    for T in (5, 600):
        held = torch.empty(T, E, device="cuda")
        out = [torch.empty(m, dtype=d, device="cuda") for m, d in
               ((T * topk, torch.int32), (T * topk, torch.float32), (E + 1, torch.int32), (T * topk, torch.int32), (T * topk, torch.int32))]
        spec = ex.RouteSpec(E, topk, n_groups=8, topk_groups=3, group_top=2)
        s = torch.cuda.Stream()

        def call(stream):
            assert ex.route(spec, held.data_ptr(), T, *[o.data_ptr() for o in out], stream=stream) == 0
        held.copy_(logits_of(1, T, E, "f32"))
        s.wait_stream(torch.cuda.current_stream())
        call(s.cuda_stream)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(torch.cuda.current_stream().cuda_stream)
        for seed in (2, 3):
            held.copy_(logits_of(seed, T, E, "f32"))
            g.replay()
            torch.cuda.synchronize()
            want, ww = eo.route(held.double().cpu().numpy(), topk, n_groups=8, topk_groups=3, group_top=2)
            assert np.array_equal(out[0].cpu().numpy().reshape(T, topk), want)
            off, g2c, c2g = eo.grouping(want, E)
            assert np.array_equal(out[2].cpu().numpy(), off) and np.array_equal(out[3].cpu().numpy(), g2c)
            assert np.array_equal(out[4].cpu().numpy(), c2g)
