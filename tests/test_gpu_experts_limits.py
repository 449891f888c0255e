"""GPU tests of the expert-layer operators at the limits of their numbers and in the kernels that only large calls reach.

Tolerances as in test_gpu_experts.py; products of small whole numbers are exact and compared bit by bit.
"""
import pytest
import torch

from test_gpu_experts import DEV, near, normal

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------ 4 bits --

def w4_values(q, k):
    return torch.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1)[..., :k].double()


@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("rows,k", [(1, 512), (3, 300), (16, 1160), (1, 4096), (20, 31)])
@pytest.mark.parametrize("zeros", [None, 15, 255])
def test_w4_of_the_largest_rows(prism, rows, k, group, zeros):
    """Every x is bf16's largest number, of one sign. Weights at their zero point give 0 exactly: the parts that cancel are
    whole multiples of x below 2^24 of them. Others, scaled down, give what they are."""
    n, parts = 40, -(-k // group)
    x = torch.full((rows, k), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16, device=DEV)
    z = None if zeros is None else torch.full((n, parts), zeros, dtype=torch.uint8, device=DEV)
    s = torch.full((n, parts), 2.0 ** -40, dtype=torch.bfloat16, device=DEV)
    if zeros != 255:
        at_zero = 0x88 if zeros is None else 0xff
        q = torch.full((n, (k + 1) // 2), at_zero, dtype=torch.uint8, device=DEV)
        assert bool((prism.gemv_w4(x, q, s, group, zeros=z, out_dtype=torch.float32) == 0).all())
    gen = torch.Generator(device=DEV).manual_seed(k)
    q = torch.randint(0, 256, (n, (k + 1) // 2), generator=gen, dtype=torch.uint8, device=DEV)
    v, zero = w4_values(q, k), 8 if zeros is None else zeros
    out = prism.gemv_w4(x, q, s, group, zeros=z, out_dtype=torch.float32)
    near(out, x.double() @ (v - zero).T * 2.0 ** -40, x.double() @ (32 + v + zero).T * 2.0 ** -40, 128 + k // 32 + 16)


@pytest.mark.parametrize("group", [32, 64, 96, 128])
@pytest.mark.parametrize("rows,k", [(1, 512), (4, 300), (16, 1160)])
@pytest.mark.parametrize("power", [-118, -126, 100, 120])
def test_w4_of_rows_of_any_size(prism, rows, k, group, power):
    """Normal values around 2^power, scales that bring the results back to ordinary numbers."""
    n, parts = 33, -(-k // group)
    x = (normal(k, rows, k).double() * 2.0 ** power).bfloat16()
    x = torch.where(x.abs() < 2.0 ** -126, 0.0, x)
    gen = torch.Generator(device=DEV).manual_seed(rows)
    q = torch.randint(0, 256, (n, (k + 1) // 2), generator=gen, dtype=torch.uint8, device=DEV)
    s = torch.full((n, parts), 2.0 ** -power, dtype=torch.float64, device=DEV).bfloat16()
    v = w4_values(q, k)
    out = prism.gemv_w4(x, q, s, group, out_dtype=torch.float32)
    near(out, x.double() @ (v - 8).T * 2.0 ** -power, x.double().abs() @ (40 + v).T * 2.0 ** -power, 128 + k // 32 + 16)
