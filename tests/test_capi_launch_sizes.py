"""CPU checks that the passes over rows refuse more threads than a launch holds (2^32 - 1, beyond which a launch runs a part
of itself with no error): every call here is turned back on the host, so the pointers are only addresses."""

import pytest

from zmoe import _lib as L

P = 0x10000  # an address on 16 bytes
BF16, F32 = 1, 0
MANY = (1 << 26) + 8  # rows of one wave each


@pytest.mark.parametrize("name,args", [
    # A, lda, K, dtype, sorted_idxs, N, fan_out, coeff, coeff_dtype, Y, ldy, stream
    ("zmoe_group", (P, 2048, 2048, BF16, P, 1 << 32, 1, None, F32, P, 2048, None)),
    # Y, gates, addend, T, k, d, dtype, out, stream
    ("zmoe_combine", (P, P, None, 1 << 32, 1, 2048, BF16, P, None)),
    # Y, grad_out, gates, inverse, T, k, d, dtype, d_gates, grouped_grad_out, stream
    ("zmoe_combine_backward", (P, P, P, P, 1 << 32, 2, 2048, BF16, P, P, None)),
    # Xe, T, k, d, dtype, add0, add1, out_dtype, out, stream
    ("zmoe_sum_k", (P, 1 << 32, 1, 2048, BF16, None, None, BF16, P, None)),
    ("zmoe_cast_f32_bf16", (P, 1 << 35, P, None)),
    # A, a_dtype, B, b_dtype, T, F, H, out, out_dtype, stream
    ("zmoe_rowwise_sum_product", (P, BF16, P, BF16, MANY, 1, 8, P, F32, None)),
    ("zmoe_rowwise_sum_product", (P, BF16, P, BF16, 1 << 62, 8, 8, P, F32, None)),
    # H, R, f, dtype, A, stream
    ("zmoe_swiglu", (P, 1 << 29, 64, BF16, P, None)),
    # dA, H, R, f, dtype, dH, ld_dh, stream
    ("zmoe_swiglu_backward", (P, P, 1 << 29, 64, BF16, P, 128, None)),
    # dA, H, R, f, row_scale, slot_of_row, dtype, dH, d_gates, stream
    ("zmoe_swiglu_backward_gates", (P, P, MANY, 8, P, P, BF16, P, P, None)),
    # X, x_stride, x_rows, rows, n, d, weight, w_dtype, eps, dtype, Y, rstd, stream
    ("zmoe_rmsnorm_rows", (P, 8, MANY, None, MANY, 8, P, BF16, 1e-6, BF16, P, P, None)),
    # d_weight, topk_prob, topk_idx, T, E, k, d_logits, ld, dtype, stream
    ("zmoe_route_topk_backward", (P, P, P, MANY, 8, 2, P, 8, BF16, None)),
    # Y, Ys, gates, addend, T, k, N, dtype, out_rows, out_total, out, stream
    ("zmoe_combine_half", (P, P, None, None, 1 << 29, 1, 64, BF16, None, 0, P, None)),
])
def test_refused(name, args):
    lib = L.load()
    assert len(args) == len(L.SIGNATURES[name][1])
    assert getattr(lib, name)(*args) == 2, lib.zmoe_last_error()
    assert b"launch" in lib.zmoe_last_error() or b"too" in lib.zmoe_last_error()
