"""Workloads of the expert-layer operators: the router, the row moves, the grouped products and the 4-bit products.

`own = False` computes each operator from elementary torch operations in 32 bits; `own = True` makes the calls of
prism_amd that a program makes. `exact` is the definition in 64 bits, group by group.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------- cases --

def listed():
    return [
        # a decoder's step with one sequence: latency is all that counts
        {"name": "route 1 token", "op": "route", "tokens": 1, "experts": 64, "k": 4, "dtype": "fp32", "renormalise": True, "empty": 0.0},
        # a prompt batch padded at its end: whole rows of -inf route nowhere
        {"name": "route prompts", "op": "route", "tokens": 16384, "experts": 256, "k": 8, "dtype": "bf16", "renormalise": True, "empty": 0.03},
        # the router's gradient in a training step, weights not renormalised
        {"name": "route gradient", "op": "route_grad", "tokens": 32768, "experts": 128, "k": 8, "dtype": "fp32", "renormalise": False, "empty": 0.0},
        # a small serving batch, rows that are no multiple of a packet
        {"name": "combine 33 tokens", "op": "combine", "tokens": 33, "experts": 40, "k": 4, "width": 2050, "dtype": "bf16", "empty": 0.1},
        # the combination's gradient in a training step
        {"name": "combine gradient", "op": "combine_grad", "tokens": 8192, "experts": 64, "k": 8, "width": 4096, "dtype": "bf16", "empty": 0.0},
        # eight decoded tokens of four experts each: every row reads its own weights
        {"name": "products 32 rows", "op": "product", "rows": 32, "spare": 0, "experts": 64, "n": 1536, "k": 2048, "out": "bf16", "skew": 0.5},
        # a ragged serving batch with an unused end of the buffer, odd widths, fp32 results
        {"name": "products ragged", "op": "product", "rows": 5003, "spare": 117, "experts": 24, "n": 1000, "k": 1048, "out": "fp32", "skew": 1.0},
        # a training step's forward products, the largest
        {"name": "products training", "op": "product", "rows": 65536, "spare": 0, "experts": 64, "n": 2048, "k": 4096, "out": "bf16", "skew": 0.3},
        # the gradients of the same step, on half of its rows
        {"name": "products grad rows", "op": "product_grad_a", "rows": 32768, "spare": 0, "experts": 32, "n": 2048, "k": 4096, "out": "bf16", "skew": 0.3},
        {"name": "products grad weights", "op": "product_grad_b", "rows": 32768, "spare": 0, "experts": 32, "n": 2048, "k": 4096, "out": "fp32", "skew": 0.3},
        # one token through a projection held in 4 bits
        {"name": "4 bits 1 row", "op": "w4", "rows": 1, "experts": 1, "n": 8192, "k": 8192, "group": 128, "zeros": False, "out": "bf16", "skew": 0.0},
        # eight tokens of four experts each, weights in 4 bits with zero points in small groups
        {"name": "4 bits 32 rows experts", "op": "w4", "rows": 32, "experts": 64, "n": 1536, "k": 2048, "group": 32, "zeros": True, "out": "fp32", "skew": 0.5},
    ]


def _log_int(rng, low, high, step=1):
    return max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step)


def draw(rng):
    op = rng.choice(["route", "route_grad", "gather", "gather_grad", "combine", "combine_grad", "product", "product",
                     "product_grad_a", "product_grad_b", "w4", "w4"])
    if op.startswith("route"):
        experts = rng.choice([8, 16, 40, 64, 128, 200, 256, 384])
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "experts": experts, "k": rng.randint(1, 8), "dtype": rng.choice(["bf16", "fp32"]),
                "renormalise": rng.random() < 0.5, "empty": rng.choice([0.0, 0.05])}
    if op in ("gather", "gather_grad", "combine", "combine_grad"):
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "experts": rng.choice([8, 40, 64, 128]), "k": rng.randint(1, 8),
                "width": _log_int(rng, 64, 4096, rng.choice([1, 2, 8, 64])), "dtype": rng.choice(["bf16", "bf16", "fp32"]), "empty": rng.choice([0.0, 0.1])}
    if op == "w4":
        experts = rng.choice([1, 1, 8, 32])
        return {"op": op, "rows": rng.choice([1, 1, 2, 3, 5, 8, 13, 16, 31, 48]), "experts": experts, "n": _log_int(rng, 128, 8192 if experts == 1 else 2048, rng.choice([1, 16, 64])),
                "k": _log_int(rng, 256, 8192 if experts == 1 else 4096, rng.choice([8, 32, 128])), "group": rng.choice([32, 64, 128]),
                "zeros": rng.random() < 0.5, "out": rng.choice(["bf16", "fp32"]), "skew": rng.choice([0.0, 0.5])}
    experts = rng.choice([4, 8, 24, 32, 64])
    step = rng.choice([1, 8, 64])
    return {"op": op, "rows": _log_int(rng, 1 if op == "product" else 256, 16384), "spare": rng.choice([0, 0, 50]), "experts": experts,
            "n": _log_int(rng, 256, 2048, step), "k": _log_int(rng, 256, 2048, step), "out": rng.choice(["bf16", "fp32"]), "skew": rng.choice([0.0, 0.3, 1.0])}


# --------------------------------------------------------------------------------------------------------- inputs --

def _group_sizes(case, rng):
    """Rows of each expert: uneven shares, as a router gives them."""
    share = np.exp(case["skew"] * rng.standard_normal(case["experts"]))
    return rng.multinomial(case["rows"], share / share.sum())


def _offsets(sizes):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).cuda()


def _logits(case, gen):
    """Router logits: normal, a few experts favoured, some tokens without any expert."""
    z = torch.randn(case["tokens"], case["experts"], generator=gen, device="cuda")
    z += 0.3 * torch.randn(case["experts"], generator=gen, device="cuda")
    gone = torch.rand(case["tokens"], generator=gen, device="cuda") < case["empty"]
    return z.masked_fill(gone[:, None], -math.inf).to(DTYPES[case.get("dtype", "fp32")])


def _plain_plan(experts, num):
    """offsets, rows, slots of the chosen experts [tokens, k]; -1: none."""
    flat = experts.reshape(-1).long()
    key = torch.where(flat < 0, num, flat)
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(num + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([torch.zeros_like(counts[:1]), torch.cumsum(counts[:num], 0)])
    place = torch.arange(flat.numel(), device=flat.device)
    rows = torch.where(place < offsets[num], order, -1)
    slots = torch.empty_like(place).scatter_(0, order, place)
    slots = torch.where(flat < 0, -1, slots).reshape(experts.shape)
    return offsets.int(), rows.int(), slots.int()


def _plain_route(logits, k, renormalise):
    z = logits.float()
    value, index = torch.sort(z, dim=1, descending=True, stable=True)
    value, index = value[:, :k], index[:, :k]
    there = value > -math.inf
    top = torch.where(there[:, :1], value[:, :1], 0.0)
    up = torch.exp(value - top)
    total = up.sum(1, keepdim=True) if renormalise else torch.exp(z - top).sum(1, keepdim=True)
    weights = torch.where(there, up / torch.where(total > 0, total, 1.0), 0.0)
    return weights, torch.where(there, index, -1).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    op = case["op"]
    if op in ("route", "route_grad"):
        state = {"case": case, "logits": _logits(case, gen)}
        if op == "route_grad":
            state["weights"], state["experts"] = _plain_route(state["logits"], case["k"], case["renormalise"])
            state["grad"] = torch.randn(case["tokens"], case["k"], generator=gen, device="cuda")
        else:  # a program's own buffers: weights, experts, offsets, rows, slots
            shape = (case["tokens"], case["k"])
            whole = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (shape, case["experts"] + 1, shape[0] * shape[1], shape)]
            state["out"] = (torch.zeros(shape, device="cuda"), *whole)
        return state
    if op in ("gather", "gather_grad", "combine", "combine_grad"):
        dtype = DTYPES[case["dtype"]]
        weights, experts = _plain_route(_logits({**case, "dtype": "fp32"}, gen), case["k"], True)
        offsets, rows, slots = _plain_plan(experts, case["experts"])
        state = {"case": case, "weights": weights, "experts": experts, "offsets": offsets, "rows": rows, "slots": slots}
        per_token = torch.randn(case["tokens"], case["width"], generator=gen, device="cuda").to(dtype)
        per_slot = torch.randn(case["tokens"] * case["k"], case["width"], generator=gen, device="cuda").to(dtype)
        if op in ("gather", "combine_grad"):
            state["tokens"] = per_token
            state["out"] = torch.zeros_like(per_slot)
        if op != "gather":
            state["slots_in"] = per_slot
        return state
    dtype = DTYPES[case["out"]]
    sizes = _group_sizes(case, rng)
    rows = case["rows"] + case.get("spare", 0)
    state = {"case": case, "offsets": _offsets(sizes), "most": int(sizes.max())}
    E, n, k = case["experts"], case["n"], case["k"]
    if op == "w4":
        groups = -(-k // case["group"])
        state["x"] = torch.randn(rows, k, generator=gen, device="cuda").bfloat16()
        state["q"] = torch.randint(0, 256, (E, n, -(-k // 2)), generator=gen, device="cuda", dtype=torch.uint8)
        state["scales"] = (0.01 * (0.5 + torch.rand(E, n, groups, generator=gen, device="cuda"))).bfloat16()
        state["zeros"] = torch.randint(4, 12, (E, n, groups), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        state["out"] = torch.zeros(rows, n, dtype=dtype, device="cuda")
        return state
    if op in ("product", "product_grad_b"):
        state["a"] = torch.randn(rows, k, generator=gen, device="cuda").bfloat16()
    if op in ("product", "product_grad_a"):
        state["b"] = (torch.randn(E, n, k, generator=gen, device="cuda") / math.sqrt(k)).bfloat16()
    if op != "product":
        state["grad"] = torch.randn(rows, n, generator=gen, device="cuda").bfloat16()
    if op != "product_grad_b":
        state["out"] = torch.zeros(rows, n if op == "product" else k, dtype=dtype, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------------- one pass --

def _padded(state, rows_of):
    """Where each row lies in a batch of groups padded to the longest, and the rows of that batch (rows_of of them
    exist; the padding points at row 0 and is masked)."""
    offsets, most = state["offsets"].long(), max(1, state["most"])
    at = offsets[:-1, None] + torch.arange(most, device=offsets.device)
    there = at < offsets[1:, None]
    row = torch.arange(rows_of, device=offsets.device)
    group = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=offsets.numel() - 2)
    back = group * most + (row - offsets[group]).clamp(max=most - 1)
    return torch.where(there, at, 0), there, back, row < offsets[-1]


def _plain_rows(state, left, right):
    """left[r] @ right[group of r], in 32 bits, for the rows of the groups; the others stay as the output has them."""
    case = state["case"]
    at, there, back, real = _padded(state, left.shape[0])
    full = torch.matmul(left.float()[at], right)
    out = full.reshape(-1, full.shape[-1])[back]
    return torch.where(real[:, None], out, state["out"].float()).to(DTYPES[case["out"]])


def _unpacked(q, k):
    return torch.stack([q & 15, q >> 4], dim=-1).reshape(*q.shape[:-1], -1)[..., :k]


def _run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "route":
        weights, experts = _plain_route(state["logits"], case["k"], case["renormalise"])
        return (weights, experts, *_plain_plan(experts, case["experts"]))
    if op == "route_grad":
        w, g, chosen = state["weights"], state["grad"], state["experts"].long()
        there = chosen >= 0
        c = (w * g).sum(1, keepdim=True)
        if case["renormalise"]:
            values, p = torch.where(there, w * (g - c), 0.0), torch.zeros(case["tokens"], case["experts"], device="cuda")
        else:
            z = state["logits"].float()
            top = z.max(1, keepdim=True).values
            p = torch.exp(z - torch.where(top > -math.inf, top, 0.0))
            total = p.sum(1, keepdim=True)
            p = -c * p / torch.where(total > 0, total, 1.0)
            values = torch.where(there, w * g, 0.0)
        return p.scatter_add_(1, chosen.clamp(min=0), values).to(state["logits"].dtype)
    if op == "gather":
        real = state["rows"] >= 0
        token = torch.div(state["rows"].clamp(min=0), case["k"], rounding_mode="floor")
        return torch.where(real[:, None], state["tokens"][token], state["out"])
    if op in ("gather_grad", "combine"):
        picked = state["slots_in"].float()[state["slots"].clamp(min=0).long()]
        w = torch.where(state["slots"] >= 0, state["weights"] if op == "combine" else 1.0, 0.0)
        return (picked * w[:, :, None]).sum(1).to(DTYPES[case["dtype"]])
    if op == "combine_grad":
        there = state["slots"] >= 0
        slots = state["slots"].clamp(min=0).long()
        up = state["tokens"].float()
        dw = torch.where(there, (state["slots_in"].float()[slots] * up[:, None]).sum(2), 0.0)
        real = state["rows"] >= 0
        flat = state["rows"].clamp(min=0).long()
        dy = up[torch.div(flat, case["k"], rounding_mode="floor")] * state["weights"].reshape(-1)[flat][:, None]
        return torch.where(real[:, None], dy, state["out"].float()).to(DTYPES[case["dtype"]]), dw
    if op == "product":
        return _plain_rows(state, state["a"], state["b"].float().transpose(1, 2))
    if op == "product_grad_a":
        return _plain_rows(state, state["grad"], state["b"].float())
    if op == "product_grad_b":
        at, there, _, _ = _padded(state, state["a"].shape[0])
        up = torch.where(there[..., None], state["grad"].float()[at], 0.0)
        return torch.matmul(up.transpose(1, 2), state["a"].float()[at]).to(DTYPES[case["out"]])
    k, group = case["k"], case["group"]
    zero = 8.0 if state["zeros"] is None else torch.repeat_interleave(state["zeros"].float(), group, dim=2)[..., :k]
    scale = torch.repeat_interleave(state["scales"].float(), group, dim=2)[..., :k]
    w = (_unpacked(state["q"], k).float() - zero) * scale
    return _plain_rows(state, state["x"], w.transpose(1, 2))


def _run_own(state):
    import prism_amd as prism

    case = state["case"]
    op = case["op"]
    if op == "route":
        r = prism.route_topk(state["logits"], case["k"], renormalise=case["renormalise"], out=state["out"])
        return r.weights, r.experts, r.offsets, r.rows, r.slots
    if op == "route_grad":
        return prism.route_topk_backward(state["grad"], state["logits"], state["weights"], state["experts"], renormalise=case["renormalise"])
    if op == "gather":
        return prism.expert_gather(state["tokens"], state["rows"], case["k"], out=state["out"])
    if op == "gather_grad":
        return prism.expert_gather_backward(state["slots_in"], state["slots"])
    if op == "combine":
        return prism.expert_combine(state["slots_in"], state["weights"], state["slots"])
    if op == "combine_grad":
        return prism.expert_combine_backward(state["tokens"], state["slots_in"], state["weights"], state["slots"], grad_y=state["out"])
    if op == "product":
        return prism.gemm_bf16_grouped(state["a"], state["b"], state["offsets"], state["out"])
    if op == "product_grad_a":
        return prism.gemm_bf16_grouped_grad_a(state["grad"], state["b"], state["offsets"], state["out"])
    if op == "product_grad_b":
        return prism.gemm_bf16_grouped_grad_b(state["grad"], state["a"], state["offsets"], out_dtype=DTYPES[case["out"]])
    return prism.gemv_w4(state["x"], state["q"], state["scales"], case["group"], zeros=state["zeros"], offsets=state["offsets"], out=state["out"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------------------------------------- work --

def work(case):
    op = case["op"]
    if op.startswith("route"):
        t, e, k = case["tokens"], case["experts"], case["k"]
        size = 2 if case["dtype"] == "bf16" else 4
        if op == "route":
            return {"bytes": t * e * size + 16 * t * k + 4 * (e + 1), "flops": 3.0 * t * e}
        return {"bytes": 2 * t * e * size + 12 * t * k, "flops": 5.0 * t * e}
    if "width" in case:
        t, k, h = case["tokens"], case["k"], case["width"]
        size = 2 if case["dtype"] == "bf16" else 4
        moved = {"gather": t + t * k, "gather_grad": t + t * k, "combine": t + t * k, "combine_grad": t + 2 * t * k}[op]
        return {"bytes": moved * h * size + 8 * t * k, "flops": {"gather": 0.0, "combine_grad": 3.0}.get(op, 2.0) * t * k * h}
    r, e, n, k = case["rows"], case["experts"], case["n"], case["k"]
    used = e if op == "product_grad_b" else e * (1 - (1 - 1 / e) ** r)
    size = 2 if case["out"] == "bf16" else 4
    flops = 2.0 * r * n * k
    if op == "w4":
        return {"bytes": used * n * (k / 2 + -(-k // case["group"]) * (3 if case["zeros"] else 2)) + 2 * r * k + size * r * n, "flops": flops}
    if op == "product":
        return {"bytes": 2 * r * k + 2 * used * n * k + size * r * n, "flops": flops}
    if op == "product_grad_a":
        return {"bytes": 2 * r * n + 2 * used * n * k + size * r * k, "flops": flops}
    return {"bytes": 2 * r * (n + k) + size * e * n * k, "flops": flops}


# ---------------------------------------------------------------------------------------------------------- exact --

def exact(case, seed):
    """The definition in 64 bits, one group or one token's list after the other."""
    s = prepare(case, seed)
    op = case["op"]
    if op in ("route", "route_grad"):
        z = s["logits"].double()
        open_ = torch.isfinite(z)
        best = torch.where(open_, z, -math.inf).amax(1, keepdim=True)
        up = torch.where(open_, torch.exp(z - torch.where(torch.isfinite(best), best, 0.0)), 0.0)
        left, picks = torch.where(open_, z, -math.inf), []
        for _ in range(case["k"]):
            top = left.amax(1, keepdim=True)
            place = torch.where(left == top, torch.arange(z.shape[1], device=z.device), z.shape[1]).amin(1, keepdim=True)
            picks.append(torch.where(top > -math.inf, place, -1))
            left = left.scatter(1, place, -math.inf)
        chosen = torch.cat(picks, 1)
        mask = torch.zeros_like(z).scatter_add_(1, chosen.clamp(min=0), (chosen >= 0).double())
        total = (up * mask if case["renormalise"] else up).sum(1, keepdim=True)
        p = up / torch.where(total > 0, total, 1.0)
        w = torch.where(chosen >= 0, p.gather(1, chosen.clamp(min=0)), 0.0)
        if op == "route":
            flat, E = chosen.reshape(-1).cpu().numpy(), case["experts"]
            lists = [np.nonzero(flat == e)[0] for e in range(E)]
            rows, slots = np.full(flat.size, -1, np.int32), np.full(flat.size, -1, np.int32)
            every = np.concatenate(lists)
            rows[: every.size] = every
            slots[every] = np.arange(every.size)
            offsets = np.concatenate([[0], np.cumsum([len(v) for v in lists])]).astype(np.int32)
            return w, chosen.int(), offsets, rows, slots.reshape(chosen.shape)
        # dL/dz_e = sum_j g_j dw_j/dz_e; w_j = p_j of a softmax over the chosen or over all
        g = torch.zeros_like(z).scatter_add_(1, chosen.clamp(min=0), torch.where(chosen >= 0, s["grad"].double(), 0.0))
        if case["renormalise"]:
            p = p * mask
        return p * (g - (p * g * mask).sum(1, keepdim=True))
    if "width" in case:
        slots, k = s["slots"].long(), case["k"]
        if op == "gather":
            out = s["out"].double()
            for j in range(k):
                ok = slots[:, j] >= 0
                out[slots[ok, j]] = s["tokens"][ok].double()
            return out
        if op in ("combine", "gather_grad"):
            out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
            for j in range(k):
                ok = slots[:, j] >= 0
                w = s["weights"][ok, j, None].double() if op == "combine" else 1.0
                out[ok] += w * s["slots_in"][slots[ok, j]].double()
            return out
        dy, dw = s["out"].double(), torch.zeros(case["tokens"], k, dtype=torch.float64, device="cuda")
        for j in range(k):
            ok = slots[:, j] >= 0
            up = s["tokens"][ok].double()
            dy[slots[ok, j]] = s["weights"][ok, j, None].double() * up
            dw[ok, j] = (up * s["slots_in"][slots[ok, j]].double()).sum(1)
        return dy, dw
    ends = s["offsets"].tolist()
    if op == "product_grad_b":
        out = torch.zeros(case["experts"], case["n"], case["k"], dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            out[e] = s["grad"][ends[e]:ends[e + 1]].double().T @ s["a"][ends[e]:ends[e + 1]].double()
        return out
    out = s["out"].double()
    for e in range(case["experts"]):
        lo, hi = ends[e], ends[e + 1]
        if lo == hi:
            continue
        if op == "product":
            out[lo:hi] = s["a"][lo:hi].double() @ s["b"][e].double().T
        elif op == "product_grad_a":
            out[lo:hi] = s["grad"][lo:hi].double() @ s["b"][e].double()
        else:
            q = s["q"][e]
            w = torch.empty(case["n"], 2 * q.shape[1], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (q % 16).double(), (q // 16).double()
            part = torch.arange(case["k"], device="cuda") // case["group"]
            z = 8.0 if s["zeros"] is None else s["zeros"][e].double()[:, part]
            out[lo:hi] = s["x"][lo:hi].double() @ ((w[:, : case["k"]] - z) * s["scales"][e].double()[:, part]).T
    return out
