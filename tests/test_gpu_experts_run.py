"""Routing, quantisation, both expert products and the combine as a mixture-of-experts layer runs them, against 64 bits stage by stage:
every stage is compared on the outputs that the stage before it left, because quantisation makes steps out of last bits."""
import importlib

import numpy as np
import pytest

import expert_ops_oracle as eo

pytestmark = pytest.mark.gpu
ex = importlib.import_module("salt-core_b200.experts")


def layer(seed, E, H, M):
    rng = np.random.default_rng(seed)

    def matrices(R, C):
        w = rng.standard_normal((E, R, C)) / np.sqrt(C)
        code, byte = zip(*(eo.mx_quantize(m) for m in w))
        return np.stack(code), np.stack(byte)
    return matrices(M, H), matrices(M, H), matrices(H, M)


@pytest.mark.parametrize("T", [1, 6, 200])
def test_layer(T):
    import torch
    E, H, M, K = 16, 256, 96, 4
    gate, up, down = layer(1, E, H, M)
    dev = [[torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (eo.mx_pack(c), b)] for c, b in (gate, up, down)]
    gu = ex.Mxfp4Weights(M, H, E, dev[0][0].data_ptr(), dev[0][1].data_ptr(), up_codes=dev[1][0].data_ptr(), up_scales=dev[1][1].data_ptr(),
                         activation="silu")
    dn = ex.Mxfp4Weights(H, M, E, dev[2][0].data_ptr(), dev[2][1].data_ptr())
    del dev                                              # the handles keep their own copies
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    logits = 2 * torch.randn(T, E, device="cuda", generator=g)
    logits[T // 2, 3:] = -torch.inf                      # a token with three experts for four places
    n = T * K

    def new(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")
    i32, u8, bf = torch.int32, torch.uint8, torch.bfloat16
    sel, w, off, g2c, c2g = new(T, K, dtype=i32), new(T, K), new(E + 1, dtype=i32), new(n, dtype=i32), new(n, dtype=i32)
    xc, xs, h = new(n, H // 2, dtype=u8), new(n, ex.scale_pitch(H), dtype=u8), new(n, M, dtype=bf)
    hc, hs, o, y = new(n, M // 2, dtype=u8), new(n, ex.scale_pitch(M), dtype=u8), new(n, H, dtype=bf), new(T, H, dtype=bf)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    spec = ex.RouteSpec(E, K, scoring="sigmoid", n_groups=4, topk_groups=2, group_top=2, scale=1.5)

    def run(stream):
        assert ex.route(spec, logits.data_ptr(), T, sel.data_ptr(), w.data_ptr(), off.data_ptr(), g2c.data_ptr(), c2g.data_ptr(), stream=stream) == 0
        assert ex.quantize(x.data_ptr(), T, H, xc.data_ptr(), xs.data_ptr(), dtype="bf16", rows=n, d_row_index=g2c.data_ptr(), index_div=K,
                           stream=stream) == 0
        assert gu.experts(xc.data_ptr(), xs.data_ptr(), off.data_ptr(), n, h.data_ptr(), y_dtype="bf16", stream=stream) == 0
        assert ex.quantize(h.data_ptr(), n, M, hc.data_ptr(), hs.data_ptr(), dtype="bf16", stream=stream) == 0
        assert dn.experts(hc.data_ptr(), hs.data_ptr(), off.data_ptr(), n, o.data_ptr(), y_dtype="bf16", stream=stream) == 0
        assert ex.combine(o.data_ptr(), n, H, c2g.data_ptr(), w.data_ptr(), T, K, y.data_ptr(), dtype="bf16", y_dtype="bf16", stream=stream) == 0

    def compare():
        torch.cuda.synchronize()
        want, ww = eo.route(logits.double().cpu().numpy(), K, scoring="sigmoid", n_groups=4, topk_groups=2, group_top=2, scale=1.5)
        assert np.array_equal(sel.cpu().numpy(), want)
        eo.close(w.double().cpu().numpy(), ww, 2.0 ** -18 * ww, "f32")
        offsets, order, back = eo.grouping(want, E)
        assert np.array_equal(off.cpu().numpy(), offsets) and np.array_equal(g2c.cpu().numpy(), order)
        live = int(offsets[-1])
        xv = eo.mx_values(*eo.mx_quantize(x.double().cpu().numpy()))[order[:live] // K]
        hv = eo.mx_values(*eo.mx_quantize(h.double().cpu().numpy()))[:live]
        gv, uv, dv = (eo.mx_values(*p) for p in (gate, up, down))
        for e in range(E):
            b, t = offsets[e], offsets[e + 1]
            if t > b:
                eo.close(h[b:t].double().cpu().numpy(), *eo.gated("silu", xv[b:t], gv[e], uv[e]), "bf16", "gate and up")
                eo.close(o[b:t].double().cpu().numpy(), *eo.product(hv[b:t], dv[e]), "bf16", "down")
        rows, wn = o.double().cpu().numpy(), w.double().cpu().numpy()
        terms = np.where(back.reshape(T, K) >= 0, wn, 0.0)[:, :, None] * rows[np.maximum(back.reshape(T, K), 0)]
        eo.close(y.double().cpu().numpy(), terms.sum(axis=1), K * 2.0 ** -24 * np.abs(terms).sum(axis=1), "bf16", "combine")

    run(s.cuda_stream)
    s.synchronize()
    compare()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        run(torch.cuda.current_stream().cuda_stream)
    x.copy_(torch.randn(T, H, device="cuda", generator=g))
    logits.copy_(2 * torch.randn(T, E, device="cuda", generator=g))
    graph.replay()
    compare()
    assert gu.status() == 0 and dn.status() == 0
