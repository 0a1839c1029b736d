"""ctypes mirror of the operators for experts outside a stack (salt_b200_route_experts, _mxfp4_*, _combine_experts in
include/salt_gpu_b200.h): routing, MXFP4 quantisation and products, and the weighted combine.

Arguments are device addresses (integers, 0 = not given) of memory on the current device; element types are "f32", "bf16" or
"f16"; row strides count elements and default to dense rows.  Functions return the C return code (0 accepted, -1 refused)."""
from __future__ import annotations

import ctypes as C

from ._lib import load_library

DTYPES = {"f32": 0, "bf16": 1, "f16": 2}
SCORINGS = {"softmax": 0, "sigmoid": 1}
ACTIVATIONS = {None: 0, "gelu_tanh": 1, "silu": 2}

_declared = None


def _lib():
    global _declared
    if _declared is None:
        lib = load_library()
        p, i, z = C.c_void_p, C.c_int, C.c_size_t
        lib.salt_b200_route_experts.argtypes = [C.POINTER(RouteSpec), p, i, z, i, p, p, p, p, p, p, p]
        lib.salt_b200_mxfp4_scale_pitch.argtypes, lib.salt_b200_mxfp4_scale_pitch.restype = [i], z
        lib.salt_b200_mxfp4_quantize.argtypes = [p, i, z, i, i, p, i, i, p, p, p, p]
        lib.salt_b200_mxfp4_weights_create.argtypes = [C.POINTER(Mxfp4Spec), p, C.POINTER(p)]
        lib.salt_b200_mxfp4_weights_destroy.argtypes = [p]
        lib.salt_b200_mxfp4_matmul.argtypes = [p, p, p, i, p, i, z, p]
        lib.salt_b200_mxfp4_experts.argtypes = [p, p, p, p, i, p, i, z, p]
        lib.salt_b200_mxfp4_status.argtypes = [p, p]
        lib.salt_b200_combine_experts.argtypes = [p, i, z, i, i, p, p, i, i, p, i, z, p]
        _declared = lib
    return _declared


class RouteSpec(C.Structure):
    """How a token's experts are chosen; scoring is "softmax" or "sigmoid"."""
    _fields_ = [("n_experts", C.c_int), ("topk", C.c_int), ("scoring", C.c_int), ("n_groups", C.c_int), ("topk_groups", C.c_int),
                ("group_top", C.c_int), ("renormalize", C.c_int), ("scale", C.c_float)]

    def __init__(self, n_experts, topk, scoring="softmax", n_groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0):
        super().__init__(n_experts, topk, SCORINGS[scoring], n_groups, topk_groups, group_top, int(renormalize), scale)


class Mxfp4Spec(C.Structure):
    _fields_ = [("rows", C.c_int), ("cols", C.c_int), ("n_experts", C.c_int), ("activation", C.c_int), ("codes", C.c_void_p),
                ("scales", C.c_void_p), ("up_codes", C.c_void_p), ("up_scales", C.c_void_p), ("expert_code_stride", C.c_size_t),
                ("expert_scale_stride", C.c_size_t), ("scale_row_stride", C.c_size_t)]


def route(spec, d_logits, rows, d_selected, d_weights, d_group_offsets=0, d_grouped_to_canonical=0, d_canonical_to_grouped=0,
          dtype="f32", row_stride=None, d_bias=0, stream=0):
    """Logits [rows][n_experts] -> selected experts and weights [rows][topk], and their grouping by expert where its three arrays
    are given."""
    return _lib().salt_b200_route_experts(C.byref(spec), d_logits, DTYPES[dtype], spec.n_experts if row_stride is None else row_stride,
                                          rows, d_bias, d_selected, d_weights, d_group_offsets, d_grouped_to_canonical,
                                          d_canonical_to_grouped, stream)


def scale_pitch(cols):
    """Bytes between the scale rows of quantised activations."""
    return int(_lib().salt_b200_mxfp4_scale_pitch(cols))


def quantize(d_x, src_rows, cols, d_codes, d_scales, dtype="f32", row_stride=None, rows=None, d_row_index=0, index_div=1, d_values=0,
             stream=0):
    """Rows to MXFP4: row i of the result is row d_row_index[i] // index_div of d_x, or row i without an index."""
    return _lib().salt_b200_mxfp4_quantize(d_x, DTYPES[dtype], cols if row_stride is None else row_stride, src_rows, cols, d_row_index,
                                           index_div, src_rows if rows is None else rows, d_codes, d_scales, d_values, stream)


def combine(d_rows, n_rows, cols, d_row_index, d_weights, tokens, topk, d_y, dtype="f32", y_dtype="f32", row_stride=None,
            y_row_stride=None, stream=0):
    """The weighted sum of each token's topk rows."""
    return _lib().salt_b200_combine_experts(d_rows, DTYPES[dtype], cols if row_stride is None else row_stride, n_rows, cols, d_row_index,
                                            d_weights, tokens, topk, d_y, DTYPES[y_dtype], cols if y_row_stride is None else y_row_stride,
                                            stream)


class Mxfp4Weights:
    """MXFP4 matrices of one or more experts, resident in HBM.  codes, scales (and up_codes, up_scales of a gated pair) are host or
    device addresses; they are copied.  activation: None, "gelu_tanh" or "silu" (read for a gated pair only)."""

    def __init__(self, rows, cols, n_experts, codes, scales, up_codes=0, up_scales=0, activation=None, expert_code_stride=0,
                 expert_scale_stride=0, scale_row_stride=0, stream=0):
        self.handle = C.c_void_p()
        self.lib = _lib()
        self.rows, self.cols, self.n_experts = rows, cols, n_experts
        spec = Mxfp4Spec(rows, cols, n_experts, ACTIVATIONS[activation] if up_codes else 0, codes, scales, up_codes, up_scales,
                         expert_code_stride, expert_scale_stride, scale_row_stride)
        if self.lib.salt_b200_mxfp4_weights_create(C.byref(spec), stream, C.byref(self.handle)) != 0:
            raise RuntimeError("salt_b200_mxfp4_weights_create failed (arguments, no sm_100 device, or out of memory)")

    def matmul(self, d_codes, d_scales, rows, d_y, y_dtype="f32", y_row_stride=None, stream=0):
        return self.lib.salt_b200_mxfp4_matmul(self.handle, d_codes, d_scales, rows, d_y, DTYPES[y_dtype],
                                               self.rows if y_row_stride is None else y_row_stride, stream)

    def experts(self, d_codes, d_scales, d_group_offsets, rows, d_y, y_dtype="f32", y_row_stride=None, stream=0):
        return self.lib.salt_b200_mxfp4_experts(self.handle, d_codes, d_scales, d_group_offsets, rows, d_y, DTYPES[y_dtype],
                                                self.rows if y_row_stride is None else y_row_stride, stream)

    def status(self, stream=0):
        """0 where every product so far is whole, -1 after one that gave up (or a refused call); reading clears it."""
        return self.lib.salt_b200_mxfp4_status(self.handle, stream)

    def close(self):
        if self.handle:
            self.lib.salt_b200_mxfp4_weights_destroy(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
