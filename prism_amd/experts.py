"""The operators of a layer of experts, over libprism_amd.so (include/prism_amd.h, "expert layers"):

  route_topk                 a token's k experts and their weights, and the plan that groups rows by expert
  expert_gather              the tokens' rows in the order of the plan
  gemm_bf16_grouped          each expert's product over its rows (bf16, fp32 accumulation)
  gemv_w4                    the same for a few rows and weights held in 4 bits
  expert_combine             the experts' rows back to their tokens, weighted

and the gradient of each as a call of its own. Like the calls in ops.py they run on torch's current stream of the
tensors' device, are asynchronous, take their outputs as arguments or allocate them, and raise ValueError / TypeError
for arguments they cannot work on. Matrices are row-major with any distance between rows (the last dimension must be
contiguous). An output that overlaps an input or another output, from a matrix' first element to its last (columns of one
buffer do), is refused. Nothing is copied to the host: the group offsets stay on the device. Nothing is recorded for
autograd: results of inputs that require gradients do not; a torch.autograd.Function around a call and its gradient call
records them.

One layer, forward:

    r = route_topk(logits, k)                                   # weights, experts, offsets, rows, slots
    xs = expert_gather(x, r.rows, k)
    h = gemm_bf16_grouped(xs, up, r.offsets, out_dtype=torch.bfloat16)
    y = gemm_bf16_grouped(act(h), down, r.offsets, out_dtype=torch.bfloat16)
    out = expert_combine(y, r.weights, r.slots)
"""
from __future__ import annotations

from operator import index
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .ops import _check

_TYPES = {torch.float32: 0, torch.bfloat16: 1}  # PRISM_TYPE_* of include/prism_amd.h


class Routing(NamedTuple):
    """route_topk's results: T tokens, k experts each, E experts in all, R = T k entries."""
    weights: "torch.Tensor"   # [T, k] fp32
    experts: "torch.Tensor"   # [T, k] int32, -1: none
    offsets: "torch.Tensor"   # [E + 1] int32: expert e's slots are offsets[e] .. offsets[e + 1] - 1
    rows: "torch.Tensor"      # [R] int32: the entry t k + j in a slot, -1: the slot is not used
    slots: "torch.Tensor"     # [T, k] int32: the slot of an entry, -1: none


def _call(function: str, name: str, tensors, *args) -> None:
    """Calls a launcher with the current stream of the tensors' device as its last argument. The launchers work on the
    current device, so another one is made current for the call. Kept short: with few tokens the host's time is what a
    layer takes."""
    device = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != device or device < 0:
            if not all(t.is_cuda for t in tensors):
                raise ValueError(f"{name}: expected a tensor in device memory (cuda), got a host tensor")
            raise ValueError(f"{name}: tensors on different devices ({tensors[0].device}, {t.device})")
    launch = getattr(_lib._lib or _lib.load(), function)
    if device == torch._C._cuda_getDevice():
        rc = launch(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = launch(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc != 0:
        _check(rc, name)


def _int(v, name: str) -> int:
    """An int argument of the C functions, which would keep only its lower 32 bits."""
    v = index(v)
    if not -0x80000000 <= v <= 0x7fffffff:
        raise ValueError(f"{name}: {v} is beyond 31 bits")
    return v


def _matrix(t: "torch.Tensor", dtypes, name: str, rows: Optional[int] = None, cols: Optional[int] = None) -> int:
    """Checks a row-major matrix; returns the elements between its rows."""
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {tuple(dtypes)}")
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (cols is not None and shape[1] != cols):
        raise ValueError(f"{name}: shape {tuple(shape)}, expected ({'any' if rows is None else rows}, {'any' if cols is None else cols})")
    n, m = shape
    if m > 0x7fffffff:
        raise ValueError(f"{name}: rows of {m} elements, beyond 31 bits")
    ld, one = t.stride()
    if one != 1 and m > 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous")
    if n <= 1 or m == 0:
        return max(m, 1)
    if ld < m:
        raise ValueError(f"{name}: rows overlap (stride {ld}, length {m})")
    return ld


def _whole(t: "torch.Tensor", dtype, name: str, *shape: int) -> None:
    """Checks a contiguous tensor of a given shape."""
    if t.dtype != dtype:
        raise TypeError(f"{name}: dtype {t.dtype} is not {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor")


def _groups(t: "torch.Tensor", dtypes, name: str, n: Optional[int] = None, k: Optional[int] = None) -> Tuple[int, int]:
    """Checks a stack of row-major matrices; returns the elements between rows and between matrices."""
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {tuple(dtypes)}")
    if t.dim() != 3 or (n is not None and t.shape[1] != n) or (k is not None and t.shape[2] != k):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected (groups, {'N' if n is None else n}, {'K' if k is None else k})")
    g, n, k = t.shape
    if max(g, n, k) > 0x7fffffff:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, beyond 31 bits")
    if k > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous")
    ld = t.stride(1) if n > 1 and k > 0 else max(k, 1)
    if ld < k:
        raise ValueError(f"{name}: rows overlap (stride {ld}, length {k})")
    one = (n - 1) * ld + k if n > 0 else 0
    stride = t.stride(0) if g > 1 and one > 0 else one
    if stride < one:
        raise ValueError(f"{name}: matrices overlap (stride {stride}, {one} elements each)")
    return ld, stride


def _out(out: Optional["torch.Tensor"], name: str, n: int, m: int, dtype, dtypes, like: "torch.Tensor") -> Tuple["torch.Tensor", int]:
    """The caller's row-major result, checked, or a new one; and the elements between its rows."""
    if out is not None:
        return out, _matrix(out, dtypes, name, n, m)
    if dtype not in _TYPES:
        raise TypeError(f"out_dtype: {dtype} not in {tuple(_TYPES)}")
    return (like.new_empty((n, m)) if dtype == like.dtype else like.new_empty((n, m), dtype=dtype)), max(m, 1)


# ------------------------------------------------------------------ router --

def route_topk(logits: "torch.Tensor", k: int, renormalise: bool = True, out: Optional[Routing] = None) -> Routing:
    """The k experts with the largest logits of every token, their softmax weights, and the plan of that choice.

    logits: [T, E] fp32 or bf16, E <= 1024, k <= min(E, 32). Equal logits go to the lower index, -inf is never chosen
    (a token with fewer than k others gets expert -1, weight 0), NaN counts as the largest. weights: the softmax over the
    chosen logits (renormalise) or over all of them; a token whose largest logit is NaN or +inf has NaN among them. The plan is expert_plan's. out: a Routing (or five tensors in its
    order) to write into.
    """
    ld = _matrix(logits, _TYPES, "logits")
    T, E = logits.shape
    k = _int(k, "k")
    if not 1 <= k <= E or k > 32:  # before anything of this size is allocated
        raise ValueError(f"route_topk: k={k}, 1 to 32 and at most the number of experts ({E}) are supported")
    if out is None:
        new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=logits.device)  # noqa: E731
        out = Routing(torch.empty((T, k), dtype=torch.float32, device=logits.device), new(T, k), new(E + 1), new(T * k), new(T, k))
    else:
        out = Routing(*out)
        _whole(out.weights, torch.float32, "weights", T, k)
        _whole(out.experts, torch.int32, "experts", T, k)
        _whole(out.offsets, torch.int32, "offsets", E + 1)
        _whole(out.rows, torch.int32, "rows", T * k)
        _whole(out.slots, torch.int32, "slots", T, k)
    need, workspace = _plan_workspace(T, k, E, logits)
    _call("prism_route_plan", "route_topk", (logits, *out), logits.data_ptr(), _TYPES[logits.dtype], ld, T, E, k, bool(renormalise), out.weights.data_ptr(),
          out.experts.data_ptr(), out.offsets.data_ptr(), out.rows.data_ptr(), out.slots.data_ptr(), 0 if workspace is None else workspace.data_ptr(), need)
    return out


def _plan_workspace(T: int, k: int, E: int, like: "torch.Tensor"):
    """Bytes of a plan's workspace, and one (none where the plan is small enough to do without)."""
    if T * k <= 4096 and E <= 512:
        return 0, None
    need = _lib.load().prism_expert_plan_workspace_bytes(T, k, E)
    return need, torch.empty(need, dtype=torch.uint8, device=like.device) if need > 16 else None


def expert_plan(experts: "torch.Tensor", num_experts: int, out=None) -> Tuple["torch.Tensor", "torch.Tensor", "torch.Tensor"]:
    """(offsets, rows, slots) of a choice of experts [T, k] int32, as in Routing: the entries t k + j in the order of their
    experts, equal experts in the order of the entries; entries outside [0, num_experts) go nowhere. An expert may occur
    twice in a token's list."""
    if experts.dim() != 2:
        raise ValueError("expert_plan: experts must be [tokens, k]")
    T, k = experts.shape
    _whole(experts, torch.int32, "experts", T, k)
    num_experts = _int(num_experts, "num_experts")
    if not 1 <= num_experts <= 1024:
        raise ValueError(f"expert_plan: {num_experts} experts, 1 to 1024 are supported")
    if out is None:
        new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=experts.device)  # noqa: E731
        out = (new(num_experts + 1), new(T * k), new(T, k))
    offsets, rows, slots = out
    _whole(offsets, torch.int32, "offsets", num_experts + 1)
    _whole(rows, torch.int32, "rows", T * k)
    _whole(slots, torch.int32, "slots", T, k)
    need, workspace = _plan_workspace(T, k, num_experts, experts)
    _call("prism_expert_plan", "expert_plan", (experts, offsets, rows, slots), experts.data_ptr(), T, k, num_experts, offsets.data_ptr(), rows.data_ptr(),
          slots.data_ptr(), workspace.data_ptr() if workspace is not None else 0, need)
    return offsets, rows, slots


def route_topk_backward(grad_weights: "torch.Tensor", logits: "torch.Tensor", weights: "torch.Tensor", experts: "torch.Tensor",
                        renormalise: bool = True, out: Optional["torch.Tensor"] = None) -> "torch.Tensor":
    """The gradient of route_topk's weights with respect to its logits (of their type), from the weights' gradient
    [T, k] fp32 and route_topk's weights and experts for these logits."""
    ld = _matrix(logits, _TYPES, "logits")
    T, E = logits.shape
    k = experts.shape[-1]
    _whole(grad_weights, torch.float32, "grad_weights", T, k)
    _whole(weights, torch.float32, "weights", T, k)
    _whole(experts, torch.int32, "experts", T, k)
    out, ldo = _out(out, "out", T, E, logits.dtype, (logits.dtype,), logits)
    _call("prism_route_topk_backward", "route_topk_backward", (logits, grad_weights, weights, experts, out), grad_weights.data_ptr(), logits.data_ptr(),
          _TYPES[logits.dtype], ld, weights.data_ptr(), experts.data_ptr(), T, E, k, bool(renormalise), out.data_ptr(), ldo)
    return out


# -------------------------------------------------------------------- rows --

def expert_gather(x: "torch.Tensor", rows: "torch.Tensor", k: int, out: Optional["torch.Tensor"] = None) -> "torch.Tensor":
    """out[s] = x[rows[s] // k] for every slot s with rows[s] >= 0; the other rows of out are left as they are (of a new
    out: undefined). x: [T, H] fp32 or bf16; rows: [R] int32, as route_topk gives it."""
    ldx = _matrix(x, _TYPES, "x")
    T, H = x.shape
    k = _int(k, "k")
    if rows.dim() != 1:
        raise ValueError("expert_gather: rows must be one-dimensional")
    _whole(rows, torch.int32, "rows", rows.shape[0])
    out, ldo = _out(out, "out", rows.shape[0], H, x.dtype, (x.dtype,), x)
    _call("prism_expert_gather", "expert_gather", (x, rows, out), x.data_ptr(), _TYPES[x.dtype], ldx, T, k, rows.data_ptr(), out.data_ptr(), ldo,
          rows.shape[0], H)
    return out


def _sum(name: str, y: "torch.Tensor", weights: Optional["torch.Tensor"], slots: "torch.Tensor", out: Optional["torch.Tensor"]) -> "torch.Tensor":
    ldy = _matrix(y, _TYPES, "y")
    R, H = y.shape
    if slots.dim() != 2:
        raise ValueError(f"{name}: slots must be [tokens, k]")
    T, k = slots.shape
    _whole(slots, torch.int32, "slots", T, k)
    if weights is not None:
        _whole(weights, torch.float32, "weights", T, k)
    out, ldo = _out(out, "out", T, H, y.dtype, (y.dtype,), y)
    _call("prism_expert_combine", name, (y, slots, out) if weights is None else (y, weights, slots, out), y.data_ptr(), _TYPES[y.dtype], ldy, R,
          0 if weights is None else weights.data_ptr(), slots.data_ptr(), T, k, out.data_ptr(), ldo, H)
    return out


def expert_gather_backward(grad: "torch.Tensor", slots: "torch.Tensor", out: Optional["torch.Tensor"] = None) -> "torch.Tensor":
    """The gradient of expert_gather's x: the sum of a token's rows of grad [R, H], slots [T, k] as route_topk gives them."""
    return _sum("expert_gather_backward", grad, None, slots, out)


def expert_combine(y: "torch.Tensor", weights: "torch.Tensor", slots: "torch.Tensor", out: Optional["torch.Tensor"] = None) -> "torch.Tensor":
    """out[t] = sum over j of weights[t, j] y[slots[t, j]] (fp32 sums, rounded once to y's type); zeros for a token without
    a slot. y: [R, H] fp32 or bf16; weights [T, k] fp32; slots [T, k] int32."""
    return _sum("expert_combine", y, weights, slots, out)


def expert_combine_backward(grad_out: "torch.Tensor", y: "torch.Tensor", weights: "torch.Tensor", slots: "torch.Tensor",
                            grad_y: Optional["torch.Tensor"] = None,
                            grad_weights: Optional["torch.Tensor"] = None) -> Tuple["torch.Tensor", "torch.Tensor"]:
    """(grad_y, grad_weights) of expert_combine: grad_y[slots[t, j]] = weights[t, j] grad_out[t] (rows of no slot are left
    as they are, of a new grad_y: undefined), grad_weights[t, j] = <grad_out[t], y[slots[t, j]]>. Every entry needs a slot
    of its own, as route_topk gives them."""
    ldy = _matrix(y, _TYPES, "y")
    R, H = y.shape
    if slots.dim() != 2:
        raise ValueError("expert_combine_backward: slots must be [tokens, k]")
    T, k = slots.shape
    _whole(slots, torch.int32, "slots", T, k)
    _whole(weights, torch.float32, "weights", T, k)
    ldd = _matrix(grad_out, (y.dtype,), "grad_out", T, H)
    grad_y, lddy = _out(grad_y, "grad_y", R, H, y.dtype, (y.dtype,), y)
    if grad_weights is None:
        grad_weights = torch.empty_like(weights)
    else:
        _whole(grad_weights, torch.float32, "grad_weights", T, k)
    _call("prism_expert_combine_backward", "expert_combine_backward", (y, grad_out, weights, slots, grad_y, grad_weights), grad_out.data_ptr(),
          _TYPES[y.dtype], ldd, y.data_ptr(), ldy, weights.data_ptr(), slots.data_ptr(), T, k, grad_y.data_ptr(), lddy, grad_weights.data_ptr(), R, H)
    return grad_y, grad_weights


# ---------------------------------------------------------------- products --

_BF16 = (torch.bfloat16,)


def gemm_bf16_grouped(A: "torch.Tensor", B: "torch.Tensor", offsets: "torch.Tensor", D: Optional["torch.Tensor"] = None,
                      out_dtype: "torch.dtype" = torch.float32) -> "torch.Tensor":
    """D[r] = A[r] @ B[g]^T for the rows offsets[g] <= r < offsets[g + 1] of every group g: gemm_bf16 group by group.

    A: [R, K] bf16, B: [groups, N, K] bf16, offsets: [groups + 1] int32 on the device (route_topk's). D: [R, N] fp32 or
    bf16 (a new one: of out_dtype); its rows outside [offsets[0], offsets[groups]) are left as they are (of a new D:
    undefined).
    """
    lda = _matrix(A, _BF16, "A")
    R, K = A.shape
    ldb, stride = _groups(B, _BF16, "B", None, K)
    G, N, _ = B.shape
    _whole(offsets, torch.int32, "offsets", G + 1)
    D, ldd = _out(D, "D", R, N, out_dtype, _TYPES, A)
    _call("prism_gemm_bf16_grouped", "gemm_bf16_grouped", (A, B, offsets, D), G, R, N, K, A.data_ptr(), lda, B.data_ptr(), ldb, stride,
          offsets.data_ptr(), D.data_ptr(), ldd, _TYPES[D.dtype])
    return D


def gemm_bf16_grouped_grad_a(dD: "torch.Tensor", B: "torch.Tensor", offsets: "torch.Tensor", dA: Optional["torch.Tensor"] = None,
                             out_dtype: "torch.dtype" = torch.float32) -> "torch.Tensor":
    """dA[r] = dD[r] @ B[g]: gemm_bf16_grouped's gradient for A. dD: [R, N] bf16; dA: [R, K], rows as for D there."""
    ldd = _matrix(dD, _BF16, "dD")
    R, N = dD.shape
    ldb, stride = _groups(B, _BF16, "B", N, None)
    G, _, K = B.shape
    _whole(offsets, torch.int32, "offsets", G + 1)
    dA, lda = _out(dA, "dA", R, K, out_dtype, _TYPES, dD)
    _call("prism_gemm_bf16_grouped_grad_a", "gemm_bf16_grouped_grad_a", (dD, B, offsets, dA), G, R, N, K, dD.data_ptr(), ldd, B.data_ptr(), ldb, stride,
          offsets.data_ptr(), dA.data_ptr(), lda, _TYPES[dA.dtype])
    return dA


def gemm_bf16_grouped_grad_b(dD: "torch.Tensor", A: "torch.Tensor", offsets: "torch.Tensor", dB: Optional["torch.Tensor"] = None,
                             out_dtype: "torch.dtype" = torch.float32) -> "torch.Tensor":
    """dB[g] = the sum over group g's rows r of dD[r]^T A[r] (an empty group: zeros): gemm_bf16_grouped's gradient for B.
    dD: [R, N] bf16, A: [R, K] bf16; dB: [groups, N, K] fp32 or bf16, written everywhere."""
    ldd = _matrix(dD, _BF16, "dD")
    R, N = dD.shape
    lda = _matrix(A, _BF16, "A", R, None)
    K = A.shape[1]
    if offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ValueError("offsets: expected groups + 1 entries")
    G = offsets.shape[0] - 1
    _whole(offsets, torch.int32, "offsets", G + 1)
    if dB is None:
        if out_dtype not in _TYPES:
            raise TypeError(f"out_dtype: {out_dtype} not in {tuple(_TYPES)}")
        dB = dD.new_empty((G, N, K), dtype=out_dtype)
    ldb, stride = _groups(dB, _TYPES, "dB", N, K)
    if dB.shape[0] != G:
        raise ValueError(f"dB: {dB.shape[0]} matrices for {G} groups")
    _call("prism_gemm_bf16_grouped_grad_b", "gemm_bf16_grouped_grad_b", (dD, A, offsets, dB), G, R, N, K, dD.data_ptr(), ldd, A.data_ptr(), lda,
          offsets.data_ptr(), dB.data_ptr(), ldb, stride, _TYPES[dB.dtype])
    return dB


_FORMS = {"forward": 0, "grad_a": 1, "grad_b": 2}  # PRISM_GROUPED_* of include/prism_amd.h


def gemm_bf16_grouped_plan(form: str, groups: int, rows: int, N: int, K: int, out_dtype: "torch.dtype" = torch.float32) -> Tuple[int, int]:
    """(rows of a tile, stages of its ring in LDS) of the kernel that a grouped product ("forward", "grad_a" or "grad_b") of
    contiguous, 16-byte aligned operands takes: (16, 0), (128, 4), (128, 2) or (256, 2); (0, 0) for an empty call."""
    import ctypes
    if form not in _FORMS:
        raise ValueError(f"gemm_bf16_grouped_plan: form {form!r} not in {tuple(_FORMS)}")
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype: {out_dtype} not in {tuple(_TYPES)}")
    tile, stages = ctypes.c_int(0), ctypes.c_int(0)
    _check(_lib.load().prism_gemm_bf16_grouped_plan(_FORMS[form], _int(groups, "groups"), _int(rows, "rows"), _int(N, "N"), _int(K, "K"), _TYPES[out_dtype],
                                                    ctypes.byref(tile), ctypes.byref(stages)), "gemm_bf16_grouped_plan")
    return tile.value, stages.value


def gemv_w4(x: "torch.Tensor", q: "torch.Tensor", scales: "torch.Tensor", group_size: int, zeros: Optional["torch.Tensor"] = None,
            offsets: Optional["torch.Tensor"] = None, out: Optional["torch.Tensor"] = None,
            out_dtype: "torch.dtype" = torch.bfloat16) -> "torch.Tensor":
    """A few rows times 4-bit weights: out[r, n] = sum over k of x[r, k] scales[n, k // G] (q[n, k] - zeros[n, k // G]).

    x: [R, K] bf16, finite. q: [N, ceil(K / 2)] uint8, two weights to a byte, the even k in the low nibble. scales: [N,
    ceil(K / G)] bf16, zeros: the same shape, uint8 (None: 8 throughout). G = group_size, a multiple of 32. With offsets
    (int32, on the device) q, scales and zeros have a leading dimension, one weight matrix per group, and row r of group g
    uses matrix g, as in gemm_bf16_grouped. out: [R, N] bf16 or fp32 (a new one: of out_dtype); rows of no group are
    left as they are. Sums are in fp32. Made for few rows a group: every 16 rows unpack the weights again.
    """
    ldx = _matrix(x, _BF16, "x")
    R, K = x.shape
    group_size = _int(group_size, "group_size")
    if group_size < 1:
        raise ValueError(f"gemv_w4: group size {group_size}")
    if q.dim() == 2:
        q = q[None]
    if scales.dim() == 2:
        scales = scales[None]
    if zeros is not None and zeros.dim() == 2:
        zeros = zeros[None]
    ldq, stride = _groups(q, (torch.uint8,), "q", None, (K + 1) // 2)
    G, N, _ = q.shape
    parts = -(-K // group_size)
    _whole(scales, torch.bfloat16, "scales", G, N, parts)
    if zeros is not None:
        _whole(zeros, torch.uint8, "zeros", G, N, parts)
    if offsets is not None:
        _whole(offsets, torch.int32, "offsets", G + 1)
    elif G != 1:
        raise ValueError(f"gemv_w4: {G} weight matrices need offsets")
    out, ldo = _out(out, "out", R, N, out_dtype, _TYPES, x)
    _call("prism_gemv_w4", "gemv_w4", [t for t in (x, q, scales, zeros, offsets, out) if t is not None], G, R, N, K, x.data_ptr(), ldx, q.data_ptr(), ldq,
          stride, scales.data_ptr(), zeros.data_ptr() if zeros is not None else 0, group_size, offsets.data_ptr() if offsets is not None else 0, out.data_ptr(),
          ldo, _TYPES[out.dtype])
    return out
