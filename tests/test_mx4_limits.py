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


# ---------------------------------------------------------------------------------------------------------------- how a product is cut
def parts_of(m, n, k):
    """from the workspace: the quantised x, and float32 sums of each part where there are several"""
    from eval_driving_safety_amd import _lib
    panels, up = -(-k // 256), lambda b: -(-b // 256) * 256
    left = _lib.load().adv_mx4_linear_workspace_bytes(m, n, k) - up(panels * m * 128) - up(panels * m * 8)
    one = 4 * m * n
    return left // one if left else 1                     # (a round-up to 256 bytes counts where a part has fewer: more than one all the same)


def test_a_product_is_cut_by_its_estimated_time():
    """parts only where they pay for their joining, whatever the number of tiles: few rows of x under many outputs are not multiplied in 256-row tiles (whose
    128 .. 255 tiles were cut in two or not at all by their number alone), a short contraction is not cut"""
    for m, n, k in ((20, 32768, 25088), (128, 32768, 4096), (2048, 4096, 4096), (2049, 4096, 25088), (3000, 4096, 25088), (4096, 4096, 25088), (4097, 4096, 25088)):
        assert parts_of(m, n, k) == 1, (m, n, k)
    for m, n, k in ((1500, 4096, 25088), (2048, 4096, 25088), (4096, 2048, 25088)):
        assert parts_of(m, n, k) == 2, (m, n, k)
    for m, n, k in ((1, 40000, 29000), (32, 4096, 25088), (301, 2048, 25088)):
        assert parts_of(m, n, k) > 2, (m, n, k)
    most = 0
    for m in (1, 17, 100, 128, 129, 300, 1000, 2047, 4096, 5000, 20000, 1 << 20):
        for n in (1, 100, 4096, 40000, 1 << 20):
            for k in (1, 2048, 25088, 1 << 20):
                if parts_of(m, n, k) > 1:
                    most = max(most, m * n)
    assert 0 < most <= 1 << 24                            # what the joining pass counts in 32 bits


CUT = [(20, 32768, 25088), (64, 40000, 9000), (100, 40000, 29000), (129, 33000, 4096), (257, 40000, 29000), (1500, 4096, 25088), (2048, 4096, 25088), (2049, 4096, 25088),
       (2300, 4100, 4096), (3000, 4096, 25088), (4097, 4096, 25088)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", CUT)
def test_hip_products_of_every_cut(m, n, k):
    """some rows of each against float64 sums of the values that the four bits hold; |off| as in the bound of a float32 sum whose additions take 32 products each"""
    from eval_driving_safety_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn(m, k, generator=gen, device="cuda").bfloat16()
    x[:, ::3] = 0
    w, b = torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5, torch.randn(n, generator=gen, device="cuda").bfloat16()
    q = ops.mx4_quantize(w)
    del w
    y = ops.mx4_linear(x, q, b, True)
    assert torch.equal(ops.mx4_linear(ops.mx4_quantize(x), q, b, True, dtype=torch.bfloat16), y)
    rows = sorted({0, 1, 31, 63, 64, 127, 128, 255, 256, m // 2, m - 2, m - 1} & set(range(m)))
    a, v = torch.tensor(O.mx4_values(x[rows].double().cpu().numpy())).cuda(), q.dequantize().double().t().contiguous()
    want, size = a @ v + b.double(), a.abs() @ v.abs() + b.double().abs()
    bound = (k / 32 + 16) * 2.0 ** -23 * size
    want = want.clamp_min(0)
    off = (y[rows].double() - want).abs() - bound - torch.finfo(torch.bfloat16).eps / 2 * (want + bound)
    assert float(off.max()) <= 0 and bool((want > 0).any())
