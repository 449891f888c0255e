"""GPU tests of the expert-layer operators at the limits of their numbers and in the kernels that only large calls reach.

Tolerances as in test_gpu_experts.py; products of small whole numbers are exact and compared bit by bit.
"""
import numpy as np
import pytest
import torch

from test_experts_plan import KERNELS
from test_gpu_experts import DEV, near, normal, table

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


# ---------------------------------------------------------------------------------------------------------- products --

@pytest.mark.parametrize("form,groups,rows,n,k,dtype,kernel", KERNELS)
def test_every_kernel_of_the_products_on_whole_numbers(prism, form, groups, rows, n, k, dtype, kernel):
    """Sums below 2^24 of whole numbers are exact in fp32 in any order, so a result is the exact sum, rounded once: the same
    bits as the library product of each group. One group is empty, the others' sizes are uneven."""
    assert prism.gemm_bf16_grouped_plan(form, groups, rows, n, k, dtype) == kernel
    rng = np.random.default_rng(rows)
    sizes = rng.multinomial(rows, [0.0] + [1 / (groups - 1)] * (groups - 1))
    offsets, ends = table(sizes), np.concatenate([[0], np.cumsum(sizes)]).tolist()
    gen = torch.Generator(device=DEV).manual_seed(rows)
    whole = lambda *shape: torch.randint(-3, 4, shape, generator=gen, device=DEV, dtype=torch.int8).bfloat16()  # noqa: E731
    a = whole(rows, k) if form != "grad_a" else None
    d = whole(rows, n) if form != "forward" else None
    b = whole(groups, n, k) if form != "grad_b" else None
    if form == "forward":
        out = prism.gemm_bf16_grouped(a, b, offsets, out_dtype=dtype)
    elif form == "grad_a":
        out = prism.gemm_bf16_grouped_grad_a(d, b, offsets, out_dtype=dtype)
    else:
        out = prism.gemm_bf16_grouped_grad_b(d, a, offsets, out_dtype=dtype)
    for g in range(groups):
        lo, hi = ends[g], ends[g + 1]
        if form == "forward":
            got, want = out[lo:hi], a[lo:hi].float() @ b[g].float().t()
        elif form == "grad_a":
            got, want = out[lo:hi], d[lo:hi].float() @ b[g].float()
        else:
            got, want = out[g], d[lo:hi].float().t() @ a[lo:hi].float()
        assert torch.equal(got, want.to(dtype)), f"group {g} of {hi - lo} rows"


class GroupedProduct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, offsets):
        import prism_amd as prism
        ctx.save_for_backward(a, b, offsets)
        return prism.gemm_bf16_grouped(a, b, offsets, out_dtype=torch.bfloat16)

    @staticmethod
    def backward(ctx, grad):
        import prism_amd as prism
        a, b, offsets = ctx.saved_tensors
        grad = grad.contiguous()
        return (prism.gemm_bf16_grouped_grad_a(grad, b, offsets, out_dtype=torch.bfloat16),
                prism.gemm_bf16_grouped_grad_b(grad, a, offsets, out_dtype=torch.bfloat16), None)


def test_gradients_are_recorded_by_a_function_around_the_calls_and_by_nothing_else(prism):
    """Whole numbers: every sum is exact and rounded once, as in the reference product by product."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    a, b, up = (torch.randint(-3, 4, s, generator=gen, device=DEV).bfloat16() for s in ((90, 64), (3, 48, 64), (90, 48)))
    a.requires_grad_()
    b.requires_grad_()
    sizes, ends = [30, 0, 60], [0, 30, 30, 90]
    assert not prism.gemm_bf16_grouped(a, b, table(sizes)).requires_grad
    GroupedProduct.apply(a, b, table(sizes)).backward(up)
    for g in range(3):
        rows = slice(ends[g], ends[g + 1])
        assert torch.equal(a.grad[rows], (up[rows].float() @ b[g].detach().float()).bfloat16())
        assert torch.equal(b.grad[g], (up[rows].float().t() @ a[rows].detach().float()).bfloat16())


def test_weights_of_a_token_whose_largest_logit_is_not_a_number(prism):
    """As documented, for both types and both sums: the choice is made, NaN is among the weights of that token and of no other."""
    z = normal(3, 5, 40)
    z[1, 7], z[2, 9], z[3, 3:5] = float("nan"), float("inf"), float("inf")
    for dtype in (torch.float32, torch.bfloat16):
        for renormalise in (True, False):
            r = prism.route_topk(z.to(dtype), 4, renormalise=renormalise)
            assert r.experts[1:4, 0].tolist() == [7, 9, 3] and int(r.experts[3, 1]) == 4
            assert r.weights.isnan().any(1).tolist() == [False, True, True, True, False]
