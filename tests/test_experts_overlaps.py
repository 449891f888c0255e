"""Outputs that overlap inputs or each other are refused by every expert-layer call, on the host and before any GPU work."""
import pytest

P = 1 << 40  # any non-null, aligned address: refusals come before a launch


@pytest.fixture(scope="module")
def lib():
    from prism_amd import _lib
    return _lib.load()


def at(i):
    """Addresses 4 GiB apart."""
    return P + (i << 32)


def overlaps(lib, call, where, pairs):
    """Moving operand `a` onto the last 4 bytes of operand `b` (bytes[b] long), for every pair, is refused."""
    for a, b, size in pairs:
        rc = call({**where, a: where[b] + size - 4})
        text = lib.prism_last_error_string().decode()
        assert rc == 1 and "overlaps" in text, (a, b, rc, text)


def test_router(lib):
    T, E, k, ld = 70, 16, 3, 20
    z, choice = 4 * ((T - 1) * ld + E), 4 * T * k
    w = {"logits": at(0), "weights": at(1), "chosen": at(2)}
    overlaps(lib, lambda o: lib.prism_route_topk(o["logits"], 0, ld, T, E, k, 1, o["weights"], o["chosen"], None), w,
             [("weights", "logits", z), ("chosen", "logits", z), ("weights", "chosen", choice)])
    w = {"logits": at(0), "weights": at(1), "chosen": at(2), "grad": at(3), "out": at(4)}
    overlaps(lib, lambda o: lib.prism_route_topk_backward(o["grad"], o["logits"], 0, ld, o["weights"], o["chosen"], T, E, k, 0, o["out"], ld, None), w,
             [("out", "logits", z), ("out", "grad", choice), ("out", "weights", choice), ("out", "chosen", choice)])


@pytest.mark.parametrize("T", [70, 5000])
def test_plans(lib, T):
    E, k, ld = 16, 3, 16
    z, entries = 4 * T * E, 4 * T * k
    need = lib.prism_expert_plan_workspace_bytes(T, k, E)
    w = {"chosen": at(0), "offsets": at(1), "rows": at(2), "slots": at(3), "ws": at(4), "logits": at(5), "weights": at(6)}
    small = T * k <= 4096
    pairs = [("offsets", "rows", entries), ("rows", "chosen", entries), ("slots", "chosen", entries), ("rows", "slots", entries), ("offsets", "chosen", entries)]
    if not small:
        pairs += [("ws", "chosen", entries), ("ws", "rows", entries), ("rows", "ws", need), ("offsets", "ws", need)]
    overlaps(lib, lambda o: lib.prism_expert_plan(o["chosen"], T, k, E, o["offsets"], o["rows"], o["slots"], o["ws"], need, None), w, pairs)
    pairs += [(a, "logits", z) for a in ("weights", "chosen", "offsets", "rows", "slots") + (() if small else ("ws",))]
    overlaps(lib, lambda o: lib.prism_route_plan(o["logits"], 0, ld, T, E, k, 1, o["weights"], o["chosen"], o["offsets"], o["rows"], o["slots"], o["ws"], need, None), w,
             pairs + [("weights", "chosen", entries), ("slots", "weights", entries)])


def test_row_moves(lib):
    T, k, R, H = 6, 2, 12, 8
    tokens, slots, entries = 4 * T * H, 4 * R * H, 4 * T * k
    w = {"x": at(0), "rows": at(1), "out": at(2)}
    overlaps(lib, lambda o: lib.prism_expert_gather(o["x"], 0, H, T, k, o["rows"], o["out"], H, R, H, None), w, [("out", "x", tokens), ("out", "rows", 4 * R)])
    w = {"y": at(0), "weights": at(1), "slots": at(2), "out": at(3)}
    overlaps(lib, lambda o: lib.prism_expert_combine(o["y"], 0, H, R, o["weights"], o["slots"], T, k, o["out"], H, H, None), w,
             [("out", "y", slots), ("out", "weights", entries), ("out", "slots", entries)])
    w = {"grad": at(0), "y": at(1), "weights": at(2), "slots": at(3), "grad_y": at(4), "grad_w": at(5)}
    overlaps(lib, lambda o: lib.prism_expert_combine_backward(o["grad"], 0, H, o["y"], H, o["weights"], o["slots"], T, k, o["grad_y"], H, o["grad_w"], R, H, None), w,
             [("grad_y", "grad", tokens), ("grad_y", "y", slots), ("grad_y", "weights", entries), ("grad_y", "slots", entries), ("grad_w", "grad", tokens),
              ("grad_w", "y", slots), ("grad_w", "weights", entries), ("grad_w", "slots", entries), ("grad_w", "grad_y", slots)])


def test_products(lib):
    G, R, N, K = 3, 10, 16, 64
    far = {"first": at(0), "second": at(1), "offsets": at(2), "out": at(3)}
    a, b, d = 2 * R * K, 2 * G * N * K, 2 * R * N
    overlaps(lib, lambda o: lib.prism_gemm_bf16_grouped(G, R, N, K, o["first"], K, o["second"], K, N * K, o["offsets"], o["out"], N, 0, None), far,
             [("out", "first", a), ("out", "second", b), ("out", "offsets", 4 * (G + 1))])
    overlaps(lib, lambda o: lib.prism_gemm_bf16_grouped_grad_a(G, R, N, K, o["first"], N, o["second"], K, N * K, o["offsets"], o["out"], K, 0, None), far,
             [("out", "first", d), ("out", "second", b), ("out", "offsets", 4 * (G + 1))])
    overlaps(lib, lambda o: lib.prism_gemm_bf16_grouped_grad_b(G, R, N, K, o["first"], N, o["second"], K, o["offsets"], o["out"], K, N * K, 0, None), far,
             [("out", "first", d), ("out", "second", a), ("first", "out", 4 * G * N * K), ("out", "offsets", 4 * (G + 1))])
    w = {"x": at(0), "q": at(1), "scales": at(2), "zeros": at(3), "offsets": at(4), "y": at(5)}
    overlaps(lib, lambda o: lib.prism_gemv_w4(G, R, N, K, o["x"], K, o["q"], K // 2, N * K // 2, o["scales"], o["zeros"], 32, o["offsets"], o["y"], N, 0, None), w,
             [("y", "x", a), ("y", "q", G * N * K // 2), ("y", "scales", 2 * G * N * K // 32), ("y", "zeros", G * N * K // 32), ("y", "offsets", 4 * (G + 1))])


def test_a_sum_without_slots_checks_its_result(lib):
    """It is written (zeros) though there is nothing to add up."""
    for out, ld, text in ((at(3) + 1, 8, "misaligned"), (at(3), 7, "row stride"), (None, 8, "null")):
        assert lib.prism_expert_combine(None, 1, 8, 0, None, at(2), 4, 2, out, ld, 8, None) == 1
        assert text in lib.prism_last_error_string().decode()
