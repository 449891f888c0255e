"""What the expert-layer operators refuse, on the host and before any GPU work (C ABI and Python mirror)."""
import pytest
import torch

import prism_amd as prism

P = 0x100000  # any non-null, aligned address: refusals come before a launch


@pytest.fixture(scope="module")
def lib():
    from prism_amd import _lib
    return _lib.load()


def refused(lib, rc, text):
    assert rc == 1 and text in lib.prism_last_error_string().decode(), lib.prism_last_error_string()


def test_grouped_products(lib):
    far = [P + (i << 32) for i in range(5)]

    def call(name="prism_gemm_bf16_grouped", groups=2, rows=8, N=16, K=32, first=far[0], ld1=32, second=far[1], ld2=32, stride=512, offsets=far[2], out=far[3], ldo=16, type=0):
        if name.endswith("grad_b"):
            return getattr(lib, name)(groups, rows, N, K, first, ld1, second, ld2, offsets, out, ldo, stride, type, None)
        return getattr(lib, name)(groups, rows, N, K, first, ld1, second, ld2, stride, offsets, out, ldo, type, None)

    for kw, text in (({"groups": -1}, "negative"), ({"rows": -1}, "negative"), ({"N": -1}, "negative"), ({"K": -3}, "negative"),
                     ({"type": 2}, "output type"), ({"type": -1}, "output type"), ({"ld1": 31}, "row stride"), ({"ld2": 31}, "row stride"),
                     ({"ldo": 15}, "row stride"), ({"stride": 511}, "stride between"), ({"first": None}, "null"), ({"second": None}, "null"),
                     ({"offsets": None}, "null"), ({"out": None}, "null"), ({"first": far[0] + 1}, "misaligned"), ({"offsets": far[2] + 2}, "misaligned"),
                     ({"out": far[3] + 2}, "misaligned"), ({"out": far[0]}, "overlaps"), ({"out": far[1] + 2000}, "overlaps"),
                     ({"out": far[2] + 8}, "overlaps"), ({"rows": 1 << 31}, "at most")):
        refused(lib, call(**kw), text)
    refused(lib, call("prism_gemm_bf16_grouped_grad_a", ld1=15, ldo=32), "row stride")
    refused(lib, call("prism_gemm_bf16_grouped_grad_a", ld1=16, ldo=31), "row stride")
    refused(lib, call("prism_gemm_bf16_grouped_grad_b", ld1=16, ldo=31), "row stride")
    refused(lib, call("prism_gemm_bf16_grouped_grad_b", ld1=16, ldo=32, stride=500), "stride between")
    refused(lib, call("prism_gemm_bf16_grouped_grad_b", ld1=16, ldo=32, out=far[1] + 400), "overlaps")
    # nothing to compute: no launch, no device needed
    for name, kw in (("prism_gemm_bf16_grouped", {"rows": 0}), ("prism_gemm_bf16_grouped", {"N": 0}), ("prism_gemm_bf16_grouped", {"groups": 0}),
                     ("prism_gemm_bf16_grouped_grad_a", {"rows": 0}), ("prism_gemm_bf16_grouped_grad_b", {"N": 0})):
        assert call(name, **kw) == 0


def test_w4(lib):
    far = [P + (i << 32) for i in range(6)]

    def call(groups=1, rows=3, N=16, K=64, x=far[0], ldx=64, q=far[1], ldq=32, stride=512, scales=far[2], zeros=None, G=32, offsets=None, y=far[4], ldy=16, type=1):
        return lib.prism_gemv_w4(groups, rows, N, K, x, ldx, q, ldq, stride, scales, zeros, G, offsets, y, ldy, type, None)

    for kw, text in (({"groups": -1}, "negative"), ({"rows": -2}, "negative"), ({"type": 3}, "output type"), ({"G": 0}, "group size"), ({"G": 16}, "group size"),
                     ({"G": 48}, "group size"), ({"G": -32}, "group size"), ({"groups": 2}, "need offsets"), ({"ldx": 63}, "row stride"), ({"ldq": 31}, "row stride"),
                     ({"ldy": 15}, "row stride"), ({"groups": 2, "offsets": far[3], "stride": 511}, "stride between"), ({"x": None}, "null"), ({"q": None}, "null"),
                     ({"scales": None}, "null"), ({"y": None}, "null"), ({"x": far[0] + 1}, "misaligned"), ({"y": far[4] + 1}, "misaligned"),
                     ({"y": far[1] + 256}, "overlaps"), ({"y": far[0]}, "overlaps")):
        refused(lib, call(**kw), text)
    assert call(rows=0) == 0 and call(N=0) == 0


def test_router(lib):
    def call(logits=P, type=0, ld=8, tokens=4, experts=8, k=2, weights=P << 1, chosen=P << 2):
        return lib.prism_route_topk(logits, type, ld, tokens, experts, k, 1, weights, chosen, None)

    for kw, text in (({"type": 2}, "logit type"), ({"tokens": -1}, "negative"), ({"experts": 0}, "experts"), ({"experts": 1025, "ld": 1025}, "experts"), ({"k": 0}, "k="),
                     ({"k": 9}, "k="), ({"experts": 64, "ld": 64, "k": 33}, "k="), ({"ld": 7}, "row stride"), ({"logits": None}, "null"), ({"weights": None}, "null"),
                     ({"logits": P + 2}, "misaligned"), ({"tokens": 1 << 31}, "31 bits")):
        refused(lib, call(**kw), text)
    assert call(tokens=0) == 0

    def back(grad=P, logits=P << 1, type=0, ld=8, w=P << 2, chosen=P << 3, tokens=4, experts=8, k=2, out=P << 4, ldo=8):
        return lib.prism_route_topk_backward(grad, logits, type, ld, w, chosen, tokens, experts, k, 0, out, ldo, None)

    for kw, text in (({"type": 9}, "logit type"), ({"k": 9}, "k="), ({"ldo": 7}, "row stride"), ({"grad": None}, "null"), ({"out": P << 1}, "overlaps"), ({"out": (P << 4) + 1}, "misaligned")):
        refused(lib, back(**kw), text)

    def plan(chosen=P, tokens=4, k=2, experts=8, offsets=P << 1, rows=P << 2, slots=P << 3, ws=None, bytes=0):
        return lib.prism_expert_plan(chosen, tokens, k, experts, offsets, rows, slots, ws, bytes, None)

    need = lib.prism_expert_plan_workspace_bytes(5000, 8, 64)
    assert need >= 64 * 4 and lib.prism_expert_plan_workspace_bytes(1, 8, 64) > 0
    for kw, text in (({"tokens": -1}, "negative"), ({"experts": 0}, "experts"), ({"k": 0}, "k="), ({"offsets": None}, "offsets"), ({"rows": None}, "rows"),
                     ({"slots": (P << 3) + 2}, "aligned"), ({"tokens": 5000, "k": 8, "experts": 64}, "workspace"),
                     ({"tokens": 5000, "k": 8, "experts": 64, "ws": P << 5, "bytes": need - 1}, "workspace"), ({"tokens": 1 << 30, "k": 4}, "31 bits")):
        refused(lib, plan(**kw), text)


def test_row_moves(lib):
    far = [P + (i << 32) for i in range(7)]
    refused(lib, lib.prism_expert_gather(far[0], 5, 8, 4, 2, far[1], far[2], 8, 8, 8, None), "element type")
    refused(lib, lib.prism_expert_gather(far[0], 0, 7, 4, 2, far[1], far[2], 8, 8, 8, None), "row stride")
    refused(lib, lib.prism_expert_gather(far[0], 0, 8, 4, 0, far[1], far[2], 8, 8, 8, None), "k=")
    refused(lib, lib.prism_expert_gather(far[0], 0, 8, 4, 2, None, far[2], 8, 8, 8, None), "rows")
    refused(lib, lib.prism_expert_gather(far[0], 0, 8, 4, 2, far[1], far[0] + 64, 8, 8, 8, None), "overlap")
    refused(lib, lib.prism_expert_gather(far[0], 0, 8, -4, 2, far[1], far[2], 8, 8, 8, None), "negative")
    refused(lib, lib.prism_expert_combine(far[0], 1, 8, 8, far[1], None, 4, 2, far[2], 8, 8, None), "slots")
    refused(lib, lib.prism_expert_combine(far[0], 1, 8, 8, far[1], far[3], 4, 2, far[0], 8, 8, None), "overlap")
    refused(lib, lib.prism_expert_combine(far[0] + 1, 1, 8, 8, far[1], far[3], 4, 2, far[2], 8, 8, None), "misaligned")
    refused(lib, lib.prism_expert_combine_backward(far[0], 1, 8, far[1], 8, far[2], far[3], 4, 2, far[1], 8, far[4], 8, 8, None), "overlaps")
    refused(lib, lib.prism_expert_combine_backward(far[0], 1, 8, far[1], 8, far[2], far[3], 4, 2, far[5], 8, None, 8, 8, None), "gradient")
    assert lib.prism_expert_gather(None, 0, 8, 4, 2, None, None, 8, 0, 8, None) == 0


def test_python_mirror():
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="device memory"):
        prism.gemm_bf16_grouped(bf(8, 32), bf(2, 16, 32), i32(3))
    with pytest.raises(ValueError, match="device memory"):
        prism.route_topk(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="device memory"):
        prism.expert_gather(bf(4, 8), i32(8), 2)
    with pytest.raises(ValueError, match="device memory"):
        prism.gemv_w4(bf(1, 64), torch.zeros(16, 32, dtype=torch.uint8), bf(16, 2), 32)
    for call, error, text in (
            (lambda: prism.gemm_bf16_grouped(torch.zeros(8, 32), bf(2, 16, 32), i32(3)), TypeError, "dtype"),
            (lambda: prism.gemm_bf16_grouped(bf(8, 32), bf(2, 16, 31), i32(3)), ValueError, "shape"),
            (lambda: prism.gemm_bf16_grouped(bf(8, 32), bf(2, 16, 32), i32(2)), ValueError, "offsets"),
            (lambda: prism.gemm_bf16_grouped(bf(8, 32), bf(2, 16, 32), torch.zeros(3, dtype=torch.int64)), TypeError, "offsets"),
            (lambda: prism.gemm_bf16_grouped(bf(32, 8).t(), bf(2, 16, 32), i32(3)), ValueError, "contiguous"),
            (lambda: prism.gemm_bf16_grouped(bf(1, 32).expand(8, 32), bf(2, 16, 32), i32(3)), ValueError, "overlap"),
            (lambda: prism.gemm_bf16_grouped(bf(8, 32), bf(1, 16, 32).expand(2, 16, 32), i32(3)), ValueError, "overlap"),
            (lambda: prism.gemm_bf16_grouped(bf(8, 32), bf(2, 16, 32), i32(3), out_dtype=torch.float16), TypeError, "out_dtype"),
            (lambda: prism.gemm_bf16_grouped(bf(8, 32), bf(2, 16, 32), i32(3), D=bf(8, 17)), ValueError, "D"),
            (lambda: prism.gemm_bf16_grouped_grad_a(bf(8, 15), bf(2, 16, 32), i32(3)), ValueError, "shape"),
            (lambda: prism.gemm_bf16_grouped_grad_b(bf(8, 16), bf(7, 32), i32(3)), ValueError, "shape"),
            (lambda: prism.gemm_bf16_grouped_grad_b(bf(8, 16), bf(8, 32), i32(3), dB=torch.zeros(3, 16, 32)), ValueError, "groups"),
            (lambda: prism.route_topk(torch.zeros(4, 8, dtype=torch.float64), 2), TypeError, "dtype"),
            (lambda: prism.expert_combine(bf(8, 8), torch.zeros(4, 3), i32(4, 2)), ValueError, "weights"),
            (lambda: prism.expert_plan(torch.zeros(4, 2, dtype=torch.int64), 8), TypeError, "experts"),
            (lambda: prism.gemv_w4(bf(1, 64), torch.zeros(16, 31, dtype=torch.uint8), bf(16, 2), 32), ValueError, "q"),
            (lambda: prism.gemv_w4(bf(1, 64), torch.zeros(16, 32, dtype=torch.uint8), bf(16, 3), 32), ValueError, "scales"),
            (lambda: prism.gemv_w4(bf(1, 64), torch.zeros(2, 16, 32, dtype=torch.uint8), bf(2, 16, 2), 32), ValueError, "offsets")):
        with pytest.raises(error, match=text):
            call()


def test_sizes_beyond_a_launch_or_31_bits(lib):
    far = [P + (i << 44) for i in range(8)]
    many = 1 << 28
    refused(lib, lib.prism_expert_gather(far[0], 1, 8, 4, 2, far[1], far[2], 8, many, 8, None), "one launch")
    refused(lib, lib.prism_expert_combine(far[0], 1, 8, 4, None, far[1], many, 2, far[2], 8, 8, None), "one launch")
    refused(lib, lib.prism_expert_combine_backward(far[0], 1, 8, far[1], 8, far[2], far[3], many >> 2, 2, far[4], 8, far[5], 8, 8, None), "one launch")
    for tokens in (many + 1, (1 << 62) + 1):
        refused(lib, lib.prism_route_topk(far[0], 1, 8, tokens, 8, 1, 1, far[1], far[2], None), "one launch" if tokens < 1 << 31 else "31 bits")
    refused(lib, lib.prism_route_topk_backward(far[0], far[1], 0, 8, far[2], far[3], many + 1, 8, 1, 0, far[4], 8, None), "one launch")
    assert lib.prism_expert_plan_workspace_bytes(1 << 20, 8, 1 << 20) == 16  # experts that no call takes
    top = 0x7fffffff
    for name in ("prism_gemm_bf16_grouped", "prism_gemm_bf16_grouped_grad_a"):
        refused(lib, getattr(lib, name)(1, 1, 1, top, far[0], top, far[1], top, top, far[2], far[3], top, 0, None), "at most")
        refused(lib, getattr(lib, name)(1, 1, top, 1, far[0], top, far[1], 1, top, far[2], far[3], top, 0, None), "at most")
        refused(lib, getattr(lib, name)(top, 1, 1, 1, far[0], 1, far[1], 1, 1, far[2], far[3], 1, 0, None), "at most")
    refused(lib, lib.prism_gemm_bf16_grouped_grad_b(1, 1, top, 1, far[0], top, far[1], 1, far[2], far[3], 1, top, 0, None), "at most")
    refused(lib, lib.prism_gemm_bf16_grouped(1 << 20, 1 << 20, 1 << 20, 8, far[0], 8, far[1], 8, 1 << 23, far[2], far[3], 1 << 20, 0, None), "too many tiles")
    refused(lib, lib.prism_gemv_w4(1, 1, top, 32, far[0], 32, far[1], 16, 0, far[2], None, 32, None, far[3], top, 1, None), "at most")
    refused(lib, lib.prism_gemv_w4(1, 1 << 20, 1 << 20, 32, far[0], 32, far[1], 16, 0, far[2], None, 32, None, far[3], 1 << 20, 1, None), "too many tiles")


def test_python_integers_are_not_cut():
    x, i32 = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: prism.route_topk(torch.zeros(4, 8), (1 << 32) + 1), lambda: prism.expert_plan(i32, (1 << 32) + 1),
                 lambda: prism.expert_gather(x, i32.view(-1), (1 << 32) + 2),
                 lambda: prism.gemv_w4(x, torch.zeros(16, 32, dtype=torch.uint8), torch.zeros(16, 1, dtype=torch.bfloat16), (1 << 32) + 32),
                 lambda: prism.gemm_bf16_grouped(torch.empty(1, 1 << 31, dtype=torch.bfloat16, device="meta"), x.view(1, 4, 64), i32.view(-1)[:2])):
        with pytest.raises(ValueError, match="31 bits"):
            call()
    for call in (lambda: prism.route_topk(torch.zeros(4, 8), 0), lambda: prism.route_topk(torch.zeros(4, 8), 9), lambda: prism.route_topk(torch.zeros(4, 64), 33),
                 lambda: prism.expert_plan(i32, 0), lambda: prism.expert_plan(i32, 1025)):
        with pytest.raises(ValueError, match="supported"):
            call()
    with pytest.raises(TypeError):
        prism.expert_gather(x, i32.view(-1), 2.0)
