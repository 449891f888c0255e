"""Which kernel a grouped product takes (no GPU needed: sizes alone decide, for 256 compute units)."""
import pytest
import torch

import prism_amd as prism

FP32, BF16 = torch.float32, torch.bfloat16

# (form, groups, rows, N, K, result, (rows of a tile, stages)): every kernel of every form, with sizes that end inside a tile.
# Tiles of 256 rows: also more tiles than 32 to a workgroup, which works them out 32 at a time.
KERNELS = [(form, *sizes, dtype, kernel) for form, sizes, kernel in (
    ("forward", (6, 90, 520, 264), (16, 0)), ("forward", (3, 700, 520, 1032), (128, 4)), ("forward", (24, 5003, 1000, 1048), (128, 2)),
    ("forward", (6, 9101, 2056, 776), (256, 2)), ("forward", (8, 6000, 2048, 2048), (256, 2)), ("forward", (4, 270000, 2048, 128), (256, 2)),
    ("grad_a", (6, 90, 520, 264), (128, 4)), ("grad_a", (16, 5000, 520, 1032), (128, 2)), ("grad_a", (6, 9101, 2056, 776), (256, 2)),
    ("grad_a", (8, 6000, 2048, 2048), (256, 2)), ("grad_a", (4, 270000, 128, 2048), (256, 2)),
    ("grad_b", (8, 700, 264, 520), (128, 4)), ("grad_b", (30, 1200, 304, 512), (128, 2)), ("grad_b", (6, 9101, 2056, 776), (256, 2)),
    ("grad_b", (8, 6000, 2048, 2048), (256, 2)), ("grad_b", (40, 4000, 4096, 4096), (256, 2))) for dtype in (FP32, BF16)]


@pytest.mark.parametrize("form,groups,rows,n,k,dtype,kernel", KERNELS)
def test_kernel_of_sizes(form, groups, rows, n, k, dtype, kernel):
    assert prism.gemm_bf16_grouped_plan(form, groups, rows, n, k, dtype) == kernel


def test_every_kernel_is_listed():
    taken = {(form, kernel) for form, *_, kernel in KERNELS}
    assert taken == {("forward", (16, 0))} | {(form, kernel) for form in ("forward", "grad_a", "grad_b") for kernel in ((128, 4), (128, 2), (256, 2))}


def test_rows_of_any_alignment_do_not_take_the_largest_tiles():
    for form in ("forward", "grad_a", "grad_b"):
        assert prism.gemm_bf16_grouped_plan(form, 6, 9101, 2051, 777)[0] == 128


def test_empty_calls_and_refusals():
    for form, sizes in (("forward", (0, 8, 8, 8)), ("forward", (2, 0, 8, 8)), ("forward", (2, 8, 0, 8)), ("grad_a", (2, 8, 8, 0)), ("grad_b", (2, 8, 0, 8))):
        assert prism.gemm_bf16_grouped_plan(form, *sizes) == (0, 0)
    assert prism.gemm_bf16_grouped_plan("grad_b", 2, 0, 8, 8) != (0, 0)  # zeros are written
    for call, error, text in ((lambda: prism.gemm_bf16_grouped_plan("grad_c", 2, 8, 8, 8), ValueError, "form"),
                              (lambda: prism.gemm_bf16_grouped_plan("forward", 2, 8, 8, 8, torch.float16), TypeError, "out_dtype"),
                              (lambda: prism.gemm_bf16_grouped_plan("forward", -1, 8, 8, 8), ValueError, "negative"),
                              (lambda: prism.gemm_bf16_grouped_plan("forward", 2, 1 << 31, 8, 8), ValueError, "31 bits"),
                              (lambda: prism.gemm_bf16_grouped_plan("forward", 1 << 40, 8, 8, 8), ValueError, "31 bits")):
        with pytest.raises(error, match=text):
            call()


def test_calls_without_a_workspace_are_those_that_need_none():
    """The Python calls know by themselves which plans need no workspace; the library must agree."""
    from prism_amd import _lib, experts
    lib, host = _lib.load(), torch.empty(0)
    for tokens in (0, 1, 64, 65, 128, 511, 512, 513, 1024, 4095, 4096, 4097, 5000):
        for k in (1, 2, 4, 8, 32):
            for num in (1, 64, 511, 512, 513, 1024):
                need, workspace = experts._plan_workspace(tokens, k, num, host)
                bytes_ = lib.prism_expert_plan_workspace_bytes(tokens, k, num)
                assert (need, workspace) == (0, None) if bytes_ == 16 else (need == bytes_ and workspace.numel() == bytes_), (tokens, k, num)
