"""Calls of the operators for experts outside a stack that the documentation does not allow are refused before any device is
asked for: these run without a GPU.  And the statements in 64 bits that the GPU tests compare with, at values worked out by hand."""
import ctypes as C
import importlib

import numpy as np
import pytest

import expert_ops_oracle as eo

ex = importlib.import_module("salt-core_b200.experts")
P = 0x1000          # an address that is never read


def route_spec(**k):
    return ex.RouteSpec(**{**dict(n_experts=64, topk=4), **k})


@pytest.mark.parametrize("bad", [dict(n_experts=0), dict(n_experts=1025), dict(topk=0), dict(topk=33), dict(topk=65),
                                 dict(n_groups=0), dict(n_groups=5), dict(n_groups=64), dict(n_groups=4, topk_groups=0),
                                 dict(n_groups=4, topk_groups=5), dict(group_top=0), dict(group_top=3),
                                 dict(n_groups=16, topk_groups=1, topk=5), dict(scale=float("nan")), dict(scale=float("inf"))])
def test_route_refuses_specs(bad):
    assert ex.route(route_spec(**bad), P, 1, P, P, P, P, P) == -1


def test_route_refuses_arguments():
    ok = dict(dtype="f32")
    s = route_spec()
    assert ex.route(s, P, -1, P, P, **ok) == -1
    assert ex.route(s, 0, 1, P, P, **ok) == -1
    assert ex.route(s, P, 1, 0, P, **ok) == -1
    assert ex.route(s, P, 1, P, 0, **ok) == -1
    assert ex.route(s, P + 2, 1, P, P, **ok) == -1                       # misaligned
    assert ex.route(s, P, 1, P, P, row_stride=63, **ok) == -1
    assert ex.route(s, P, 1, P, P, d_group_offsets=P, **ok) == -1        # part of a grouping
    assert ex.route(s, P, 1, P, P, d_grouped_to_canonical=P, d_canonical_to_grouped=P, **ok) == -1
    assert ex.route(s, P, 1 << 23, P, P, **ok) == -1                     # too many selections
    for i in range(6):                                                   # misaligned tables
        p = [P + 2 if i == j else P for j in range(6)]
        assert ex.route(s, P, 1, *p[:5], d_bias=p[5], **ok) == -1
    assert ex._lib().salt_b200_route_experts(C.byref(s), P, 3, 64, 1, 0, P, P, 0, 0, 0, 0) == -1
    assert ex._lib().salt_b200_route_experts(None, P, 0, 64, 1, 0, P, P, 0, 0, 0, 0) == -1
    assert ex.route(s, 0, 0, 0, 0, **ok) == 0                            # no rows, no grouping: nothing to do


def test_quantize_refuses_arguments():
    ok = dict(src_rows=4, cols=64, d_codes=P, d_scales=P)
    for bad in (dict(cols=0), dict(cols=16), dict(cols=48), dict(cols=131072 + 32), dict(src_rows=-1), dict(rows=-1), dict(rows=5),
                dict(row_stride=63), dict(row_stride=65), dict(d_codes=0), dict(d_scales=0), dict(d_codes=P + 8),
                dict(d_scales=P + 8), dict(d_values=P + 4), dict(d_row_index=P, index_div=0),
                dict(d_row_index=P + 1)):
        assert ex.quantize(P, **{**ok, **bad}) == -1, bad
    assert ex.quantize(0, **ok) == -1 and ex.quantize(P + 4, **ok) == -1
    assert ex.quantize(P, dtype="bf16", row_stride=68, **ok) == -1       # rows that begin on 8 bytes
    assert ex._lib().salt_b200_mxfp4_quantize(P, 3, 64, 4, 64, 0, 1, 4, P, P, 0, 0) == -1
    assert ex.quantize(0, 0, 64, 0, 0) == 0
    assert [ex.scale_pitch(c) for c in (32, 512, 544, 2816)] == [16, 16, 32, 96] == [eo.scale_pitch(c) for c in (32, 512, 544, 2816)]


def test_weights_refuse_specs():
    ok = dict(rows=8, cols=64, n_experts=2, codes=P, scales=P)
    for bad in (dict(rows=0), dict(rows=(1 << 24) + 1), dict(cols=0), dict(cols=33), dict(cols=131072 + 32), dict(n_experts=0),
                dict(n_experts=1025), dict(codes=0), dict(scales=0), dict(up_codes=P), dict(up_scales=P),
                dict(up_codes=P, up_scales=P), dict(scale_row_stride=1), dict(expert_code_stride=8 * 32 - 1),
                dict(expert_scale_stride=15)):
        with pytest.raises(RuntimeError):
            ex.Mxfp4Weights(**{**ok, **bad})


def test_products_without_a_handle():
    lib = ex._lib()
    assert lib.salt_b200_mxfp4_matmul(0, P, P, 1, P, 0, 64, 0) == -1
    assert lib.salt_b200_mxfp4_experts(0, P, P, P, 1, P, 0, 64, 0) == -1
    assert lib.salt_b200_mxfp4_weights_destroy(0) == -1 and lib.salt_b200_mxfp4_status(0, 0) == -1


def test_combine_refuses_arguments():
    ok = dict(d_rows=P, n_rows=8, cols=64, d_row_index=P, d_weights=P, tokens=2, topk=4, d_y=P)
    for bad in (dict(n_rows=-1), dict(cols=0), dict(tokens=-1), dict(topk=0), dict(topk=33), dict(d_rows=0), dict(d_weights=0),
                dict(d_y=0), dict(row_stride=63), dict(y_row_stride=63), dict(d_rows=P + 2), dict(d_y=P + 1),
                dict(d_row_index=P + 1), dict(d_weights=P + 2)):
        assert ex.combine(**{**ok, **bad}) == -1, bad
    assert ex.combine(**{**ok, "tokens": 0, "d_y": 0}) == 0


def test_statement_of_the_format():
    x = np.zeros((1, 64))
    x[0, :10] = [4.0, -6.9, 7.9, 2.5, 3.5, 5.0, 0.25, 0.75, -0.2, 1.75]     # largest in [4, 8): a unit of 1
    code, byte = eo.mx_quantize(x)
    assert byte.tolist() == [[127, 0]]
    assert code[0, :10].tolist() == [6, 15, 7, 4, 6, 6, 0, 2, 8, 4] and not code[0, 10:].any()
    v = eo.mx_values(code, byte)
    assert v[0, :10].tolist() == [4.0, -6.0, 6.0, 2.0, 4.0, 4.0, 0.0, 1.0, -0.0, 2.0]
    assert (eo.mx_unpack(eo.mx_pack(code)) == code).all()
    x[0, 40] = np.nan
    code, byte = eo.mx_quantize(x)
    assert byte.tolist() == [[127, 255]] and np.isnan(eo.mx_values(code, byte)[0, 32:]).all()


def test_statement_of_routing():
    l = np.array([[1.0, 3.0, 3.0, 0.0, np.nan, -np.inf, 2.0, 3.0]])
    ids, w = eo.route(l, 2)
    assert ids.tolist() == [[1, 2]] and np.allclose(w, 0.5)
    ids, w = eo.route(l, 8)
    assert ids.tolist() == [[0, 1, 2, 3, 6, 7, -1, -1]] and w[0, 6:].tolist() == [0.0, 0.0] and abs(w.sum() - 1) < 1e-12
    # groups {1 3}, {3 0}, {nan -inf}, {2 3}: the best keys are 3, 3, none, 3, so the lower two groups stay
    ids, _ = eo.route(l, 2, n_groups=4, topk_groups=2)
    assert ids.tolist() == [[1, 2]]
    ids, _ = eo.route(l, 1, scoring="sigmoid", bias=[0, 0, 0, 0, 9, 9, 9, 0])
    assert ids.tolist() == [[6]]
    offsets, g2c, c2g = eo.grouping(np.array([[1, 3], [0, -1], [1, 2]]), 4)
    assert offsets.tolist() == [0, 1, 3, 4, 5] and g2c.tolist() == [2, 0, 4, 5, 1, -1] and c2g.tolist() == [1, 4, 0, -1, 2, 3]
