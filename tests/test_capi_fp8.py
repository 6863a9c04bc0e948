"""CPU checks of what the e4m3 and norm_residual entry points of the C ABI refuse: every call here is turned back on the
host, before any launch, so the pointers are only addresses."""

import ctypes

import pytest

from zmoe import _lib as L

OK, NULL, SHAPE, DTYPE, ALIGN, WORKSPACE = 0, 1, 2, 3, 4, 5
P = 0x10000  # an address on 16 bytes
BF16, F32 = 1, 0


def call(name, *args):
    return getattr(L.load(), name)(*args)


def refused(name, good, changes):
    """good: the arguments of a call that would launch; each change of one or more of them is refused with its code."""
    for code, change in changes:
        args = list(good)
        for i, v in change.items():
            args[i] = v
        assert call(name, *args) == code, (name, change, L.load().zmoe_last_error())


@pytest.mark.parametrize("K,pitch", [(1, 4), (128, 4), (512, 4), (513, 8), (7168, 56), ((1 << 30) - 1, 1 << 23)])
def test_scale_pitch(K, pitch):
    got = ctypes.c_int64()
    assert call("zmoe_fp8_scale_pitch", K, ctypes.addressof(got)) == OK and got.value == pitch


def test_scale_pitch_refusals():
    got = ctypes.c_int64()
    for K in (0, -1, 1 << 30):
        assert call("zmoe_fp8_scale_pitch", K, ctypes.addressof(got)) == SHAPE
    assert call("zmoe_fp8_scale_pitch", 4, None) == NULL


def test_quantize_rows_refusals():
    # X, x_stride, x_rows, rows, row_div, row_scale, n, K, dtype, Q, S, stream
    good = (P, 64, 8, None, 1, None, 8, 64, BF16, P, P, None)
    refused("zmoe_fp8_quantize_rows", good, [
        (DTYPE, {8: 7}), (SHAPE, {6: -1}), (SHAPE, {7: 0}), (SHAPE, {7: 1 << 30}), (SHAPE, {6: 1 << 31}), (SHAPE, {1: 63}),
        (SHAPE, {4: 0}), (SHAPE, {2: -1}), (SHAPE, {2: 7}), (NULL, {9: None}), (NULL, {10: None}), (NULL, {0: None}),
        (ALIGN, {9: P + 8}), (ALIGN, {10: P + 2}),
        (SHAPE, {6: (1 << 31) - 2, 2: (1 << 31) - 1, 7: 256, 1: 256}),  # more blocks than a launch has
    ])
    assert call("zmoe_fp8_quantize_rows", None, 64, 0, None, 1, None, 0, 64, BF16, None, None, None) == OK  # no rows


def test_quantize_weight_refusals():
    # W, w_stride_e, w_stride_n, E, N, K, dtype, Q, S, Qt, St, stream
    good = (P, 64 * 32, 64, 2, 32, 64, F32, P, P, P, P, None)
    refused("zmoe_fp8_quantize_weight", good, [
        (DTYPE, {6: -1}), (SHAPE, {3: 0}), (SHAPE, {3: 65536}), (SHAPE, {4: 0}), (SHAPE, {5: 0}), (SHAPE, {2: 63}),
        (SHAPE, {1: -1}), (SHAPE, {4: 128 * 65535 + 1}), (NULL, {0: None}), (NULL, {7: None}), (NULL, {8: None}),
        (NULL, {9: None}), (NULL, {10: None}), (ALIGN, {7: P + 4}), (ALIGN, {8: P + 1}), (ALIGN, {9: P + 4}),
        (ALIGN, {10: P + 2}),
    ])


@pytest.mark.parametrize("half", [False, True])
def test_product_refusals(half):
    # Xq, Xs, M, Wq, Ws, idxs, offsets, K, N, E, k, x_grouped, y_grouped, (out_dtype, Y, y_stride | Y, Ys), stream
    head = (P, P, 16, P, P, P, P, 256, 64, 4, 2, 0, 0)
    name = "zmoe_fp8_scatter2scatter" + ("_half" if half else "")
    good = head + ((P, P, None) if half else (BF16, P, 64, None))
    refused(name, good, [
        (SHAPE, {2: -1}), (SHAPE, {7: 0}), (SHAPE, {8: 0}), (SHAPE, {9: 0}), (SHAPE, {9: 1025}), (SHAPE, {10: 0}),
        (SHAPE, {2: 1 << 31}), (SHAPE, {2: 1 << 30, 10: 2}), (NULL, {6: None}), (NULL, {5: None}),
        (NULL, {0: None}), (NULL, {1: None}), (NULL, {3: None}), (NULL, {4: None}), (ALIGN, {0: P + 8}), (ALIGN, {1: P + 2}),
        (ALIGN, {3: P + 1}), (ALIGN, {4: P + 2}),
        (SHAPE, {8: 1 << 23}),            # one expert's weights past 2 GiB
        (SHAPE, {2: 1 << 23, 10: 1}),     # gathered rows past 2 GiB
        (SHAPE, {7: 1 << 24, 2: 1, 8: 1}),  # a tile's rows past 2 GiB
    ])
    if half:
        refused(name, good, [(NULL, {13: None}), (NULL, {14: None}), (ALIGN, {13: P + 8})])
    else:
        refused(name, good, [(DTYPE, {13: 5}), (SHAPE, {15: 63}), (NULL, {14: None}), (ALIGN, {14: P + 1}),
                             (ALIGN, {13: F32, 14: P + 2})])
    # without offsets: one weight, rows in order
    for change in ({9: 2, 11: 1, 12: 1, 10: 1}, {9: 1, 11: 0, 12: 1}, {9: 1, 11: 1, 12: 0}):
        args = list(good)
        for i, v in {6: None, **change}.items():
            args[i] = v
        assert call(name, *args) == NULL
    empty = list(good)
    empty[2] = 0
    assert call(name, *empty) == OK


def test_few_rows_refusals():
    # X, x_stride, M, Wq, Ws, K, N, dtype, Y, y_stride, stream
    good = (P, 256, 16, P, P, 256, 64, BF16, P, 64, None)
    refused("zmoe_fp8_linear_few", good, [
        (DTYPE, {7: 5}), (SHAPE, {2: 17}), (SHAPE, {2: -1}), (SHAPE, {5: 0}), (SHAPE, {5: 252}), (SHAPE, {1: 248}), (SHAPE, {1: 260}),
        (SHAPE, {7: F32, 1: 258}), (SHAPE, {6: 0}), (SHAPE, {9: 63}), (NULL, {0: None}), (NULL, {3: None}), (NULL, {4: None}),
        (NULL, {8: None}), (ALIGN, {0: P + 8}), (ALIGN, {3: P + 8}), (ALIGN, {4: P + 2}), (ALIGN, {8: P + 1}),
        (SHAPE, {6: 1 << 23, 9: 1 << 23}),
    ])
    assert call("zmoe_fp8_linear_few", None, 256, 0, None, None, 256, 64, BF16, None, 64, None) == OK


def test_glu_refusals():
    # Xq, Xs, T, W1q, W1s, idxs, offsets, d, f, E, k, Aq, As, stream
    good = (P, P, 16, P, P, P, P, 256, 64, 4, 2, P, P, None)
    refused("zmoe_fp8_glu_w1_forward", good, [
        (SHAPE, {2: -1}), (SHAPE, {7: 0}), (SHAPE, {8: 0}), (SHAPE, {8: 1 << 29}), (SHAPE, {9: 1025}), (SHAPE, {10: 0}),
        (SHAPE, {2: 1 << 30, 10: 2}), (NULL, {5: None}), (NULL, {6: None}), (NULL, {11: None}), (NULL, {12: None}),
        (ALIGN, {11: P + 8}), (ALIGN, {12: P + 2}), (NULL, {3: None}), (ALIGN, {3: P + 8}), (SHAPE, {8: 1 << 22}),
    ])


def test_combine_half_refusals():
    # Y, Ys, gates, addend, T, k, N, dtype, out_rows, out_total, out, stream
    good = (P, P, P, None, 4, 2, 64, BF16, None, 4, P, None)
    refused("zmoe_combine_half", good, [
        (DTYPE, {7: 9}), (SHAPE, {4: -1}), (SHAPE, {5: 0}), (SHAPE, {6: 0}), (SHAPE, {4: 1 << 30, 5: 2}), (SHAPE, {9: -1}),
        (NULL, {0: None}), (NULL, {1: None}), (NULL, {10: None}), (ALIGN, {0: P + 4}),
        (SHAPE, {4: (1 << 31) - 2, 5: 1, 6: 1 << 20}),  # more elements than a launch has
    ])


def test_norm_residual_refusals():
    # R, r_stride, r_dtype, Y, y_stride, y_dtype, n, d, w_post, w_next, w_dtype, gate, gate_kind, gate_stride, gate_dtype,
    # scale_ptr, scale, eps, R_out, X, rstd_post, rstd_next, stream
    good = (P, 64, F32, P, 64, BF16, 8, 64, P, P, BF16, P, 3, 64, BF16, None, 1.0, 1e-6, P, P, P, P, None)
    refused("zmoe_norm_residual", good, [
        (DTYPE, {2: 2}), (DTYPE, {5: 2}), (DTYPE, {10: 2}), (DTYPE, {14: 2}), (SHAPE, {6: -1}), (SHAPE, {7: 0}),
        (SHAPE, {7: 32769, 1: 32769, 4: 32769, 13: 32769}), (SHAPE, {12: 4}), (SHAPE, {12: -1}), (SHAPE, {12: 0}),
        (SHAPE, {11: None}), (SHAPE, {1: 63}), (SHAPE, {4: 63}), (SHAPE, {13: 63}), (NULL, {8: None, 9: None}),
        (NULL, {0: None}), (NULL, {3: None}), (NULL, {18: None}), (NULL, {19: None}), (NULL, {9: None}),
    ])


def test_norm_residual_backward_refusals():
    n, d = 8, 64
    need = call("zmoe_norm_residual_backward_workspace_bytes", n, d)
    assert need > 0
    for bad in ((-1, 64), (8, 0), (8, 32769)):
        assert call("zmoe_norm_residual_backward_workspace_bytes", *bad) == 0
    # dR_out, dX, R, r_stride, r_dtype, Y, y_stride, y_dtype, n, d, w_post, w_next, w_dtype, gate, gate_kind, gate_stride,
    # gate_dtype, scale_ptr, scale, rstd_post, rstd_next, dR, dY, dw_post, dw_next, dgate, dscale, ws, ws_bytes, stream
    good = (P, P, P, d, F32, P, d, BF16, n, d, P, P, BF16, None, 0, 0, BF16, P, 1.0, P, P, P, P, P, P, None, P, P, need, None)
    refused("zmoe_norm_residual_backward", good, [
        (DTYPE, {4: 2}), (SHAPE, {9: 0}), (SHAPE, {3: 63}), (NULL, {10: None, 11: None}), (NULL, {2: None}), (NULL, {5: None}),
        (NULL, {21: None}), (NULL, {22: None}), (NULL, {19: None}), (NULL, {20: None}), (NULL, {11: None}),
        (NULL, {17: None}), (WORKSPACE, {27: None}), (WORKSPACE, {28: need - 1}), (ALIGN, {27: P + 8}), (SHAPE, {13: P}),
    ])


@pytest.mark.parametrize("d", [1, 512, 2048, 4096, 7168, 32768])
def test_norm_residual_workspace_grows_with_the_rows_it_serves(d):
    """Never less for more rows: a workspace of the largest batch serves every smaller one."""
    sizes = [call("zmoe_norm_residual_backward_workspace_bytes", n, d) for n in range(0, 20000, 37)]
    assert sizes == sorted(sizes)
