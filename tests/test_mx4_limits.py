"""MXFP4 matrices (csrc/mx4.hip): what is refused because of its size, the oracle where its scale is at its end, the product's plans."""
import numpy as np
import pytest
import torch

from oracle import oracle_np as O


def test_sizes_that_the_kernels_do_not_index_are_refused_with_the_reason():
    from eval_driving_safety_amd import ops
    ops._fits(1 << 20, 1 << 20, "x")
    for rows, cols in (((1 << 20) + 1, 1), (1, (1 << 20) + 1)):
        with pytest.raises(ValueError, match=r"x: .*at most 2\*\*20 rows"):
            ops._fits(rows, cols, "x")


@pytest.mark.gpu
def test_hip_matrices_of_too_many_rows_are_refused_with_the_reason():
    from eval_driving_safety_amd import ops
    tall = torch.zeros(((1 << 10) + 1, 1 << 10, 4), dtype=torch.bfloat16, device="cuda")
    w = ops.mx4_quantize(torch.zeros((4, 4), dtype=torch.bfloat16, device="cuda"))
    for call in (lambda: ops.mx4_quantize(tall), lambda: ops.mx4_linear(tall, w), lambda: ops.mx4_linear_dgrad(tall, w)):
        with pytest.raises(ValueError, match="take it in parts"):
            call()
    assert ops.mx4_linear(tall[:-1], w).shape == (1 << 10, 1 << 10, 4)


def test_oracle_at_the_end_of_the_scales_range():
    """blocks whose scale is held at 2^-127: what lies on that scale's grid is kept, what lies under its first midpoint is gone"""
    kept = np.ldexp(np.array([[6.0, 3.0, 1.5, 0.5, -2.0]]), -127).astype(np.float32)
    assert np.array_equal(O.mx4_values(kept), kept.astype(np.float64))
    for e in (-130, -140, -149):                       # the largest: 6 * 2^-130 = 0.75 * 2^-127, a tie that goes to 1 * 2^-127
        x = np.ldexp(np.array([[6.0, 2.0, 1.5, 0.5, -4.0]]), e).astype(np.float32)
        want = np.ldexp(np.array([[1.0, 0.0, 0.0, 0.0, -0.5]]), -127) if e == -130 else np.zeros((1, 5))
        assert np.array_equal(O.mx4_values(x), want), e
