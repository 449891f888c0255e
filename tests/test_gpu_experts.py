"""GPU tests of the expert-layer operators against plain fp64 implementations.

Tolerances, derived: u = 2^-24 is fp32's half step. A sum of n terms in fp32, in any order and with an addition off by up
to a whole step, is off by at most 2 n u times the sum of the terms' magnitudes. A bf16 result adds half a bf16 step,
2^-8 of its value. Whole numbers are equal.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
STEP = 2.0 ** -23
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}
TYPES = [torch.float32, torch.bfloat16]


def near(got, want, mag, terms):
    """|got - want| <= terms * 2^-23 * mag + half a step of got's type, element by element; NaN nowhere."""
    got64 = got.double()
    bad = ~((got64 - want).abs() <= terms * STEP * mag + HALF[got.dtype] * want.abs() * (1 + 1e-6) + 1e-38)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((got64 - want).abs().max())}"


def fenced(values, start=0, stride=None, fill=math.nan):
    """A matrix as a view of a buffer whose other elements are `fill`: first element number `start`, rows `stride` apart."""
    n, m = values.shape
    stride = m if stride is None else stride
    buf = torch.full((start + n * stride + 64,), fill, dtype=values.dtype, device=DEV)
    view = buf[start:start + n * stride].view(n, stride)[:, :m]
    view.copy_(values)
    return view


def table(sizes, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(sizes)]), dtype=torch.int32, device=DEV)


def normal(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


# ---------------------------------------------------------------------------------------------------------- products --

def grouped_case(prism, sizes, n, k, dtype, seed=0, first=0, behind=0, start=0, pad=0, forms="dab"):
    """All three products of one set of groups, rows of no group holding NaN (in) and -7 (out)."""
    rows = first + sum(sizes) + behind
    offsets = table(sizes, first)
    ends = offsets.tolist()
    a, d = normal(seed, rows, k).bfloat16(), normal(seed + 1, rows, n).bfloat16()
    for t in (a, d):
        t[:first] = math.nan
        t[rows - behind:] = math.nan
    b = (normal(seed + 2, len(sizes), n, k) / 4).bfloat16()
    a, d = fenced(a, start, k + pad), fenced(d, start, n + pad)
    b = fenced(b.view(len(sizes) * n, k), start, k + pad)
    b = torch.as_strided(b, (len(sizes), n, k), (n * (k + pad), k + pad, 1), b.storage_offset())
    real = torch.zeros(rows, dtype=torch.bool, device=DEV)
    real[first:ends[-1]] = True
    if "d" in forms:
        out = fenced(torch.full((rows, n), -7.0, dtype=dtype, device=DEV), start, n + pad, fill=-7.0)
        assert prism.gemm_bf16_grouped(a, b, offsets, out) is out
        assert bool((out[~real] == -7).all()) and bool((out._base == -7).sum() >= out._base.numel() - real.sum() * n)
        for g, size in enumerate(sizes):
            x, w = a[ends[g]:ends[g + 1]].double(), b[g].double()
            near(out[ends[g]:ends[g + 1]], x @ w.T, x.abs() @ w.abs().T, k + 8)
    if "a" in forms:
        out = fenced(torch.full((rows, k), -7.0, dtype=dtype, device=DEV), start, k + pad, fill=-7.0)
        prism.gemm_bf16_grouped_grad_a(d, b, offsets, out)
        assert bool((out[~real] == -7).all()) and bool((out._base == -7).sum() >= out._base.numel() - real.sum() * k)
        for g, size in enumerate(sizes):
            x, w = d[ends[g]:ends[g + 1]].double(), b[g].double()
            near(out[ends[g]:ends[g + 1]], x @ w, x.abs() @ w.abs(), n + 8)
    if "b" in forms:
        out = prism.gemm_bf16_grouped_grad_b(d, a, offsets, out_dtype=dtype)
        for g, size in enumerate(sizes):
            x, y = d[ends[g]:ends[g + 1]].double(), a[ends[g]:ends[g + 1]].double()
            near(out[g], x.T @ y, x.abs().T @ y.abs(), size + 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [0, 0], [3, 0, 1, 0], [127, 128, 129, 0, 1], [0, 300, 5, 64], [16, 17, 15, 1, 0, 33, 2, 8], [700], [255, 256, 257, 513]],
                         ids=lambda s: "+".join(map(str, s)))
@pytest.mark.parametrize("n,k", [(128, 128), (264, 72), (1, 1), (33, 75), (520, 1160)], ids=lambda v: str(v))
def test_grouped_products(prism, sizes, n, k, dtype):
    grouped_case(prism, sizes, n, k, dtype, seed=sum(sizes) + n + k, first=3, behind=5)


@pytest.mark.parametrize("sizes,n,k,start,pad", [([40, 0, 130], 136, 200, 8, 8), ([40, 0, 130], 136, 200, 1, 0), ([40, 0, 130], 136, 200, 0, 3), ([40, 9], 135, 201, 3, 5),
                                                 ([300, 270], 256, 512, 8, 64), ([300, 270], 256, 512, 4, 0), ([2, 1, 0, 3], 512, 1024, 0, 24), ([2, 1, 0, 3], 513, 1023, 1, 1)])
def test_grouped_products_strides_and_alignments(prism, sizes, n, k, start, pad):
    for dtype in TYPES:
        grouped_case(prism, sizes, n, k, dtype, seed=n + k + pad, first=1, behind=130, start=start, pad=pad)


@pytest.mark.parametrize("sizes,n,k", [([900, 1100, 40, 700], 1024, 1536), ([513] * 12, 768, 512), ([2048, 0, 2500], 2048, 640), ([130] * 40, 520, 328),
                                       ([3000, 5000], 1500, 1032), ([60] * 64, 512, 256), ([20] * 100, 384, 640),
                                       ([2500, 1300, 0, 3100, 700, 1], 1536, 512), ([1700, 2300, 1800, 2222, 257], 1400, 520), ([129] * 33 + [900], 1288, 2056)], ids=lambda v: str(len(v)) if isinstance(v, list) else str(v))
def test_grouped_products_with_more_tiles_than_workgroups(prism, sizes, n, k):
    grouped_case(prism, sizes, n, k, torch.bfloat16, seed=n, behind=7)
    grouped_case(prism, sizes, n, k, torch.float32, seed=n + 1)


@pytest.mark.parametrize("sizes,n,k,start,pad", [([257] * 9, 1301, 523, 1, 0), ([1] * 20 + [900, 0, 640], 1000, 1048, 0, 0), ([40] * 30, 305, 513, 3, 1), ([900, 800], 1160, 1096, 8, 8)],
                         ids=lambda v: str(len(v)) if isinstance(v, list) else str(v))
def test_grouped_products_of_two_workgroups_to_a_unit(prism, sizes, n, k, start, pad):
    for dtype in TYPES:
        grouped_case(prism, sizes, n, k, dtype, seed=n + k, first=2, behind=9, start=start, pad=pad)


def test_grouped_products_many_groups(prism):
    rng = np.random.default_rng(4)
    grouped_case(prism, list(rng.integers(0, 4, 1000)), 64, 128, torch.float32, seed=9)
    grouped_case(prism, [0] * 70 + [5] + [0] * 100 + [200] + [0], 128, 64, torch.bfloat16, seed=10)


def test_grouped_products_without_depth_or_rows(prism):
    zero = prism.gemm_bf16_grouped(torch.empty(6, 0, dtype=torch.bfloat16, device=DEV), torch.empty(2, 5, 0, dtype=torch.bfloat16, device=DEV), table([4, 2]))
    assert zero.shape == (6, 5) and bool((zero == 0).all())
    a, b = torch.empty(0, 32, dtype=torch.bfloat16, device=DEV), torch.randn(2, 16, 32, device=DEV).bfloat16()
    assert prism.gemm_bf16_grouped(a, b, table([0, 0])).shape == (0, 16)
    grad = prism.gemm_bf16_grouped_grad_b(torch.empty(0, 16, dtype=torch.bfloat16, device=DEV), a, table([0, 0]))
    assert grad.shape == (2, 16, 32) and bool((grad == 0).all())


def test_group_tables_with_wrong_contents_stay_inside(prism):
    """Entries below 0, beyond the rows and out of order are cut: results mean nothing, the fences stay."""
    a, b = fenced(normal(1, 64, 64).bfloat16()), normal(2, 4, 64, 64).bfloat16()
    for entries in ([-5, 10, 1000, 2 ** 31 - 1, 3], [64, 0, 64, 0, 64], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31, 7]):
        offsets = torch.tensor(entries, dtype=torch.int32, device=DEV)
        for call, first in ((prism.gemm_bf16_grouped, a), (prism.gemm_bf16_grouped_grad_a, a)):
            out = fenced(torch.zeros(64, 64, device=DEV), 64, fill=-7.0)
            call(first, b, offsets, out)
            assert bool((out._base[:64] == -7).all()) and bool((out._base[64 + 64 * 64:] == -7).all())
        assert prism.gemm_bf16_grouped_grad_b(a, a, offsets).shape == (4, 64, 64)
        q = torch.zeros(4, 64, 32, dtype=torch.uint8, device=DEV)
        out = fenced(torch.zeros(64, 64, device=DEV), 64, fill=-7.0)
        prism.gemv_w4(a, q, torch.ones(4, 64, 2, dtype=torch.bfloat16, device=DEV), 32, offsets=offsets, out=out)
        assert bool((out._base[:64] == -7).all()) and bool((out._base[64 + 64 * 64:] == -7).all())
    torch.cuda.synchronize()


def test_grouped_products_beyond_32_bit_offsets(prism):
    """The last rows of 2.4e9 elements of A, and the last of 4.3 GB of weight matrices."""
    rows, k, n = 300_000, 8192, 40
    a = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV)
    a[-70:] = normal(1, 70, k).bfloat16()
    d = torch.zeros(rows, n, dtype=torch.bfloat16, device=DEV)
    d[-70:] = normal(2, 70, n).bfloat16()
    offsets = torch.tensor([rows - 70, rows - 60, rows], dtype=torch.int32, device=DEV)
    b = normal(3, 2, n, k).bfloat16()
    out = prism.gemm_bf16_grouped(a, b, offsets)
    x, w = a[-60:].double(), b[1].double()
    near(out[-60:], x @ w.T, x.abs() @ w.abs().T, k + 8)
    grad = prism.gemm_bf16_grouped_grad_b(d, a, offsets)
    y = d[-60:].double()
    near(grad[1], y.T @ x, y.abs().T @ x.abs(), 68)
    back = prism.gemm_bf16_grouped_grad_a(d, b, offsets)
    near(back[-60:], y @ w, y.abs() @ w.abs(), n + 8)
    # one long group: the K loop of grad_b passes 2 GiB of A
    one = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    grad = prism.gemm_bf16_grouped_grad_b(d, a, one)
    x, y = a[-70:].double(), d[-70:].double()
    near(grad[0], y.T @ x, y.abs().T @ x.abs(), 78)
    del a, d, out, back
    big = torch.zeros(560, 1024, 4096, dtype=torch.bfloat16, device=DEV)
    big[-1] = normal(4, 1024, 4096).bfloat16()
    sizes = [0] * 559 + [20]
    a = normal(5, 20, 4096).bfloat16()
    near(prism.gemm_bf16_grouped(a, big, table(sizes)), a.double() @ big[-1].double().T, a.double().abs() @ big[-1].double().abs().T, 4104)


def test_grouped_products_are_bilinear(prism):
    """Differences: on small whole numbers every product and sum is exact, so that <dD, f(A + E, B) - f(A, B)> equals
    <dA, E>, and the same for B."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    whole = lambda *s: torch.randint(-4, 5, s, generator=gen, device=DEV).bfloat16()  # noqa: E731
    sizes, n, k = [37, 0, 130, 5], 136, 96
    rows, offsets = sum(sizes), table(sizes)
    a, ea, b, eb, d = whole(rows, k), whole(rows, k), whole(4, n, k), whole(4, n, k), whole(rows, n)
    f = lambda x, w: prism.gemm_bf16_grouped(x, w, offsets).double()  # noqa: E731
    grad_a, grad_b = prism.gemm_bf16_grouped_grad_a(d, b, offsets).double(), prism.gemm_bf16_grouped_grad_b(d, a, offsets).double()
    assert float(((f(a + ea, b) - f(a, b)) * d.double()).sum()) == float((grad_a * ea.double()).sum())
    assert float(((f(a, b + eb) - f(a, b)) * d.double()).sum()) == float((grad_b * eb.double()).sum())


# ------------------------------------------------------------------------------------------------------------ 4 bits --

def w4_case(prism, sizes, n, k, group, zeros, dtype, seed=0, start=0, pad=0, offsets=True, behind=0):
    G, rows = len(sizes), sum(sizes) + behind
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = fenced(normal(seed, rows, k).bfloat16(), start, k + pad)
    packed = (k + 1) // 2
    q = torch.randint(0, 256, (G, n, packed + pad), generator=gen, dtype=torch.uint8, device=DEV)[:, :, :packed]
    parts = -(-k // group)
    s = (0.1 + torch.rand(G, n, parts, generator=gen, device=DEV)).bfloat16()
    z = torch.randint(0, 16, (G, n, parts), generator=gen, dtype=torch.uint8, device=DEV) if zeros else None
    out = fenced(torch.full((rows, n), -7.0, dtype=dtype, device=DEV), start, n + pad, fill=-7.0)
    if offsets:
        prism.gemv_w4(x, q, s, group, zeros=z, offsets=table(sizes), out=out)
    else:
        prism.gemv_w4(x, q[0], s[0], group, zeros=None if z is None else z[0], out=out)
    at = torch.arange(k, device=DEV) // group
    values = torch.stack([q & 15, q >> 4], -1).reshape(G, n, -1)[:, :, :k].double()
    zs = torch.full_like(values, 8.0) if z is None else z.double()[:, :, at]
    ss = s.double()[:, :, at]
    lo = 0
    for g, size in enumerate(sizes):
        v = x[lo:lo + size].double()
        # the parts (16 + q) x and (16 + z) x are summed apart: their magnitudes count. Terms: at most 128 in a part,
        # K / 32 parts, 8 wavefronts, and the roundings of the combination
        mag = v.abs() @ ((32 + values[g] + zs[g]) * ss[g]).T
        near(out[lo:lo + size], v @ ((values[g] - zs[g]) * ss[g]).T, mag, 128 + k // 32 + 16)
        lo += size
    assert bool((out[lo:] == -7).all()) and bool((out._base == -7).sum() >= out._base.numel() - lo * n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("rows,n,k", [(1, 256, 512), (3, 100, 1000), (16, 33, 257), (17, 48, 1160), (64, 65, 2048), (130, 20, 31), (1, 1, 1), (2, 16, 128), (33, 16, 4224)])
def test_w4_dense(prism, rows, n, k, group, zeros, dtype):
    w4_case(prism, [rows], n, k, group, zeros, dtype, seed=rows + n + k, offsets=False)


@pytest.mark.parametrize("sizes", [[1, 0, 2, 0, 1], [0], [17, 0, 16, 33, 1], [1] * 70, [0, 0, 100]], ids=lambda s: str(len(s)))
@pytest.mark.parametrize("n,k,group,start,pad", [(64, 256, 64, 0, 0), (50, 300, 32, 1, 3), (96, 1024, 128, 8, 16)])
def test_w4_groups(prism, sizes, n, k, group, start, pad):
    w4_case(prism, sizes, n, k, group, True, torch.float32, seed=n + k, start=start, pad=pad, behind=3)
    w4_case(prism, sizes, n, k, group, False, torch.bfloat16, seed=n + k, start=start, pad=pad)


def test_w4_beyond_32_bit_offsets(prism):
    """The last of 4.3 GB of packed weights."""
    G, n, k = 130, 4096, 16384
    q = torch.zeros(G, n, k // 2, dtype=torch.uint8, device=DEV)
    q[-1] = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV)
    s = torch.ones(G, n, k // 128, dtype=torch.bfloat16, device=DEV)
    x = normal(2, 2, k).bfloat16()
    out = prism.gemv_w4(x, q, s, 128, offsets=table([0] * (G - 1) + [2]), out_dtype=torch.float32)
    values = torch.stack([q[-1] & 15, q[-1] >> 4], -1).reshape(n, k).double()
    near(out, x.double() @ (values - 8).T, x.double().abs() @ (values + 40).T, 128 + k // 32 + 16)


# ------------------------------------------------------------------------------------------------------------ router --

def plain_choice(logits, k, renormalise):
    """Experts and weights in 64 bits on the host, one token at a time."""
    z = logits.double().cpu().numpy()
    T, E = z.shape
    experts, weights = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        order = sorted((e for e in range(E) if z[t, e] != -math.inf), key=lambda e: (-z[t, e], e))[:k]
        experts[t, :len(order)] = order
        if order:
            up = np.exp(z[t] - z[t, order[0]])
            weights[t, :len(order)] = up[order] / (up[order].sum() if renormalise else up.sum())
    return torch.from_numpy(weights).to(DEV), torch.from_numpy(experts).to(DEV)


def plain_plan(experts, num):
    flat = experts.reshape(-1).cpu().numpy()
    order = [i for e in range(num) for i in np.nonzero(flat == e)[0]]
    rows, slots = np.full(flat.size, -1, np.int32), np.full(flat.size, -1, np.int32)
    rows[:len(order)] = order
    slots[order] = np.arange(len(order))
    offsets = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(num)])]).astype(np.int32)
    return [torch.from_numpy(v).to(DEV) for v in (offsets, rows, slots.reshape(experts.shape))]


@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 64, 4), (7, 8, 8), (33, 40, 5), (100, 65, 1), (513, 128, 8), (70, 256, 16), (70, 257, 32), (40, 512, 8), (9, 1024, 32), (2100, 17, 2)])
def test_route(prism, tokens, experts, k, dtype, renormalise):
    z = normal(tokens + experts, tokens, experts)
    z = (z * 4).round() / 4 if tokens % 2 else z  # many equal logits
    z[:, ::3] -= 30.0
    if experts > 2:
        z[tokens // 2] = -math.inf          # a token without experts
        z[tokens // 3, 1:] = -math.inf      # and one with a single one
        z[0, 0], z[0, 1] = 0.0, -0.0
    z = fenced(z.to(dtype), 3, experts + tokens % 3)
    r = prism.route_topk(z, k, renormalise=renormalise)
    weights, chosen = plain_choice(z, k, renormalise)
    assert torch.equal(r.experts, chosen)
    # exp is off by at most two steps and its argument by half a step of up to 40; the sum adds at most 32 steps
    assert bool(((r.weights.double() - weights).abs() <= 80 * STEP * weights + 1e-38).all())
    for got, want in zip(r[2:], plain_plan(chosen, experts)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("tokens,k,num", [(1, 1, 1), (300, 3, 5), (4096, 1, 512), (513, 8, 64), (5000, 8, 100), (700, 6, 1024), (20000, 8, 1), (40001, 4, 777), (0, 4, 8)])
def test_plan_of_any_choice(prism, tokens, k, num):
    """Experts twice in a token's list, entries outside [0, num), one expert for nearly everything, no tokens at all."""
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    chosen = torch.randint(-2, num + 2, (tokens, k), generator=gen, device=DEV, dtype=torch.int32)
    chosen[torch.rand(tokens, k, generator=gen, device=DEV) < 0.3] = num // 2
    for got, want in zip(prism.expert_plan(chosen, num), plain_plan(chosen, num)):
        assert torch.equal(got, want)


def test_route_nan_and_infinity(prism):
    z = torch.tensor([[1.0, math.nan, 3.0, -math.nan], [math.inf, 0.0, math.inf, -math.inf], [0.0, 1.0, -math.inf, -math.inf]], device=DEV)
    r = prism.route_topk(z, 3)
    assert r.experts.tolist() == [[1, 3, 2], [0, 2, 1], [1, 0, -1]]
    assert bool(r.weights[:2].isnan().any(1).all()) and float(r.weights[2, 2]) == 0 and abs(float(r.weights[2].sum()) - 1) < 1e-6
    assert r.offsets.tolist() == [0, 2, 5, 7, 8] and r.rows.tolist() == [3, 7, 0, 5, 6, 2, 4, 1, -1]


@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (5, 8, 8), (33, 40, 5), (300, 128, 8), (70, 257, 32), (6, 1024, 4), (2, 7, 3)])
def test_route_gradient(prism, tokens, experts, k, dtype, renormalise):
    z = normal(experts, tokens, experts)
    if experts > 2:
        z[tokens // 2] = -math.inf
        z[0, 1:] = -math.inf
    z = z.to(dtype)
    g = normal(7, tokens, k)
    r = prism.route_topk(z, k, renormalise=renormalise)
    got = prism.route_topk_backward(g, fenced(z, 1, experts + 1), r.weights, r.experts, renormalise=renormalise)
    zz = z.double()
    there = r.experts >= 0
    at = r.experts.clamp(min=0).long()
    mask = torch.zeros_like(zz).scatter_add_(1, at, there.double())
    up = torch.where(zz > -math.inf, torch.exp(zz - zz.masked_fill(zz == -math.inf, -1e30).amax(1, keepdim=True).clamp(min=-1e29)), 0.0)
    p = (up * mask if renormalise else up)
    p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    full = torch.zeros_like(zz).scatter_add_(1, at, torch.where(there, g.double(), 0.0))
    c = (p * full * mask).sum(1, keepdim=True)
    # every factor within some 40 steps of its value (the weights' bound above), g - c within that of |g| + sum w |g|
    near(got, p * (full - c), p * (full.abs() + (p * full.abs()).sum(1, keepdim=True)), 200 + k)


def test_route_gradient_against_differences(prism):
    """Central differences of the definition in 64 bits, away from ties: off by O(h^2)."""
    for renormalise in (True, False):
        z = normal(3, 6, 12).double()
        g = normal(4, 6, 4).double()
        _, chosen = plain_choice(z, 4, renormalise)
        at = chosen.long()

        def value(zz):
            up = torch.exp(zz)
            picked = up.gather(1, at)
            return (g * picked / (picked if renormalise else up).sum(1, keepdim=True)).sum(1)

        h, want = 1e-5, torch.zeros_like(z)
        for e in range(z.shape[1]):
            step = torch.zeros_like(z)
            step[:, e] = h
            want[:, e] = (value(z + step) - value(z - step)) / (2 * h)
        z32 = z.float()
        r = prism.route_topk(z32, 4, renormalise=renormalise)
        got = prism.route_topk_backward(g.float(), z32, r.weights, r.experts, renormalise=renormalise)
        assert float((got.double() - want).abs().max()) <= 1e-6 + 1e-9  # fp32 values of size 1: 8 steps, and h^2


# -------------------------------------------------------------------------------------------------------------- rows --

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,width,start,pad", [(1, 1, 1, 0, 0), (5, 4, 2050, 0, 0), (33, 3, 64, 0, 0), (100, 8, 4096, 0, 0), (7, 33, 100, 4, 4), (64, 2, 513, 1, 2), (9, 5, 1000, 2, 6)])
def test_rows_to_the_experts_and_back(prism, tokens, k, width, start, pad, dtype):
    experts = 11
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    chosen = torch.randint(-1, experts, (tokens, k), generator=gen, device=DEV, dtype=torch.int32)
    if tokens > 2:
        chosen[tokens // 2] = -1
    weights = normal(2, tokens, k)
    _, rows, slots = prism.expert_plan(chosen, experts)
    R = tokens * k
    used = rows >= 0
    x = fenced(normal(3, tokens, width).to(dtype), start, width + pad)
    out = fenced(torch.full((R, width), -7.0, dtype=dtype, device=DEV), start, width + pad, fill=-7.0)
    prism.expert_gather(x, rows, k, out)
    assert torch.equal(out[used], x[(rows[used] // k).long()]) and bool((out[~used] == -7).all())
    y = normal(4, R, width).to(dtype)
    y[~used] = math.nan  # behind the last slot
    y = fenced(y, start, width + pad)
    picked = torch.where((slots >= 0)[..., None], y[slots.clamp(min=0).long()].double(), 0.0)
    for got, w in ((prism.expert_combine(y, weights, slots), weights.double()), (prism.expert_gather_backward(y, slots), torch.ones(tokens, k, device=DEV, dtype=torch.float64))):
        near(got, (picked * w[..., None]).sum(1), (picked * w[..., None]).abs().sum(1), k + 2)
    up = fenced(normal(5, tokens, width).to(dtype), start, width + pad)
    grad_y = fenced(torch.full((R, width), -7.0, dtype=dtype, device=DEV), start, width + pad, fill=-7.0)
    _, grad_w = prism.expert_combine_backward(up, y, weights, slots, grad_y=grad_y)
    dots = picked * up.double()[:, None]
    near(grad_w, dots.sum(2), dots.abs().sum(2), width + 8)
    flat = rows[used].long()
    want = weights.reshape(-1)[flat, None].double() * up.double()[flat // k]
    near(grad_y[used], want, want.abs(), 1)
    assert bool((grad_y[~used] == -7).all()) and bool((grad_y._base == -7).sum() >= grad_y._base.numel() - used.sum() * width)


def test_row_moves_with_wrong_entries_stay_inside(prism):
    x = fenced(normal(1, 4, 16))
    rows = torch.tensor([0, 8, -1, 2 ** 31 - 1, -2 ** 31, 7], dtype=torch.int32, device=DEV)
    out = fenced(torch.full((6, 16), -7.0, device=DEV), 16, fill=-7.0)
    prism.expert_gather(x, rows, 2, out)
    assert torch.equal(out[0], x[0]) and torch.equal(out[5], x[3]) and bool((out[1:5] == -7).all())
    y = fenced(normal(2, 6, 16))
    slots = torch.tensor([[0, 6], [2 ** 31 - 1, -1], [-2 ** 31, 5]], dtype=torch.int32, device=DEV)
    assert torch.equal(prism.expert_gather_backward(y, slots), torch.stack([y[0], torch.zeros_like(y[0]), y[5]]))
    grad_y = fenced(torch.full((6, 16), -7.0, device=DEV), 16, fill=-7.0)
    _, grad_w = prism.expert_combine_backward(x[:3], y, torch.ones(3, 2, device=DEV), slots, grad_y=grad_y)
    assert torch.equal(grad_y[0], x[0]) and torch.equal(grad_y[5], x[2]) and bool((grad_y[1:5] == -7).all())
    assert bool((grad_w.reshape(-1)[[1, 2, 3, 4]] == 0).all())


def test_row_moves_and_router_beyond_32_bit_offsets(prism):
    """Rows 2^30 + 8 elements apart: the last of four begins beyond 2^31 elements."""
    far = (1 << 30) + 8

    def spread(values):
        view = torch.as_strided(torch.empty(3 * far + values.shape[1], dtype=values.dtype, device=DEV), tuple(values.shape), (far, 1))
        view.copy_(values)
        return view

    x, y = normal(1, 4, 264).bfloat16(), normal(2, 4, 264).bfloat16()
    rows = torch.tensor([3, 1, 0, 2], dtype=torch.int32, device=DEV)
    slots = torch.tensor([[2], [1], [3], [0]], dtype=torch.int32, device=DEV)
    w = normal(3, 4, 1)
    out = spread(torch.zeros_like(x))
    prism.expert_gather(spread(x), rows, 1, out)
    assert torch.equal(out, x[rows.long()])
    far_y, order = spread(y), slots[:, 0].long()
    prism.expert_combine(far_y, w, slots, out)
    near(out, y[order].double() * w.double(), (y[order].double() * w.double()).abs(), 2)
    grad_y, grad_w = prism.expert_combine_backward(spread(x), far_y, w, slots, grad_y=out)
    near(grad_w[:, 0], (x.double() * y[order].double()).sum(1), (x.double() * y[order].double()).abs().sum(1), 264 + 8)
    near(grad_y[order], x.double() * w.double(), (x.double() * w.double()).abs(), 1)
    logits = normal(4, 4, 64).bfloat16()
    want, got = prism.route_topk(logits, 3), prism.route_topk(spread(logits), 3)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    up = normal(5, 4, 3)
    grad = prism.route_topk_backward(up, spread(logits), got.weights, got.experts, renormalise=False, out=spread(torch.zeros_like(logits)))
    assert torch.equal(grad, prism.route_topk_backward(up, logits, want.weights, want.experts, renormalise=False))


@pytest.mark.parametrize("dtype,slots_of_all,width", [(torch.bfloat16, 13001, 8197), (torch.float32, 6700, 8192)])
def test_rows_beyond_the_caches(prism, dtype, slots_of_all, width):
    tokens, k = 301, 3
    gen = torch.Generator(device=DEV).manual_seed(width)
    slots = torch.randperm(slots_of_all, generator=gen, device=DEV)[:tokens * k].int().view(tokens, k).contiguous()
    slots[5], slots[6, 1] = -1, -1
    used = torch.zeros(slots_of_all, dtype=torch.bool, device=DEV)
    used[slots[slots >= 0].long()] = True
    y = normal(1, slots_of_all, width).to(dtype)
    y[~used] = math.nan
    up, w = normal(2, tokens, width).to(dtype), normal(3, tokens, k)
    picked = torch.where((slots >= 0)[..., None], y[slots.clamp(min=0).long()].double(), 0.0)
    near(prism.expert_combine(y, w, slots), (picked * w.double()[..., None]).sum(1), (picked * w.double()[..., None]).abs().sum(1), k + 2)
    grad_y, grad_w = prism.expert_combine_backward(up, y, w, slots, grad_y=torch.full_like(y, -7.0))
    dots = picked * up.double()[:, None]
    near(grad_w, dots.sum(2), dots.abs().sum(2), width + 8)
    want = w.double()[..., None] * up.double()[:, None]
    near(grad_y[slots[slots >= 0].long()], want[slots >= 0], want[slots >= 0].abs(), 1)
    assert bool((grad_y[~used] == -7).all())


def test_no_tokens_or_no_slots(prism):
    none = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device=DEV)  # noqa: E731
    r = prism.route_topk(none(0, 8), 2)
    assert r.weights.shape == (0, 2) and bool((r.offsets == 0).all())
    assert prism.route_topk_backward(r.weights, none(0, 8), r.weights, r.experts).shape == (0, 8)
    assert prism.expert_gather(none(0, 16), r.rows, 2).shape == (0, 16)
    assert prism.expert_combine(none(0, 16), r.weights, r.slots).shape == (0, 16)
    nowhere = torch.full((3, 2), -1, dtype=torch.int32, device=DEV)
    assert bool((prism.expert_combine(none(0, 16), normal(1, 3, 2), nowhere) == 0).all())
    grad_y, grad_w = prism.expert_combine_backward(normal(1, 3, 16), none(0, 16), normal(1, 3, 2), nowhere)
    assert grad_y.shape == (0, 16) and bool((grad_w == 0).all())
    y = prism.gemv_w4(none(3, 0, dtype=torch.bfloat16), none(5, 0, dtype=torch.uint8), none(5, 0, dtype=torch.bfloat16), 32)
    assert y.shape == (3, 5) and bool((y == 0).all())
    assert prism.gemv_w4(none(0, 64, dtype=torch.bfloat16), none(5, 32, dtype=torch.uint8), none(5, 2, dtype=torch.bfloat16), 32).shape == (0, 5)


# ----------------------------------------------------------------------------------------------- together, as in use --

def layer(prism, x, router, up, down, k):
    """One layer of experts and its gradients for the gradient x of its output; everything a training step needs."""
    logits = x.float() @ router
    r = prism.route_topk(logits, k)
    xs = prism.expert_gather(x, r.rows, k)
    xs = torch.where((r.rows >= 0)[:, None], xs, 0.0).to(x.dtype)
    h = prism.gemm_bf16_grouped(xs, up, r.offsets, out_dtype=torch.bfloat16)
    y = prism.gemm_bf16_grouped(h, down, r.offsets, out_dtype=torch.bfloat16)
    out = prism.expert_combine(y, r.weights, r.slots)
    grad_y, grad_w = prism.expert_combine_backward(x, y, r.weights, r.slots)
    grad_down = prism.gemm_bf16_grouped_grad_b(grad_y, h, r.offsets)
    grad_h = prism.gemm_bf16_grouped_grad_a(grad_y, down, r.offsets, out_dtype=torch.bfloat16)
    grad_up = prism.gemm_bf16_grouped_grad_b(grad_h, xs, r.offsets)
    grad_xs = prism.gemm_bf16_grouped_grad_a(grad_h, up, r.offsets, out_dtype=torch.bfloat16)
    grad_logits = prism.route_topk_backward(grad_w, logits, r.weights, r.experts)
    return out, grad_down, grad_up, prism.expert_gather_backward(grad_xs, r.slots), grad_logits, r


def layer_inputs(seed, tokens=96, width=128, inner=200, experts=6):
    x = normal(seed, tokens, width).bfloat16()
    return x, normal(seed + 1, width, experts) / 8, (normal(seed + 2, experts, inner, width) / 12).bfloat16(), (normal(seed + 3, experts, width, inner) / 14).bfloat16()


def test_a_layer_forward_and_backward(prism):
    """Against autograd of the same layer in 64 bits. Roundings to bf16 on the way (h, y, grad_y, grad_h, grad_xs, the results), half a step of 2^-8
    each and independent in the elements: every result is a sum over at least 48 such terms, so that its relative error in the 2-norm
    stays below four roundings' worth, 4 * 2^-8."""
    x, router, up, down = layer_inputs(11)
    out, grad_down, grad_up, grad_x, grad_logits, r = layer(prism, x, router, up, down, 2)
    logits = (x.float() @ router).double().requires_grad_()
    xx, uu, dd = (t.double().requires_grad_() for t in (x, up, down))
    w = torch.softmax(logits.gather(1, r.experts.long()), 1)
    want = torch.zeros_like(xx)
    for j in range(2):
        e = r.experts[:, j].long()
        want = want + w[:, j, None] * torch.matmul(dd[e], torch.matmul(uu[e], xx[:, :, None]))[:, :, 0]
    (want * x.double()).sum().backward()
    for got, ref in ((out, want.detach()), (grad_down, dd.grad), (grad_up, uu.grad), (grad_x, xx.grad), (grad_logits, logits.grad)):
        assert float((got.double() - ref).norm() / ref.norm()) <= 4 * 2.0 ** -8


def test_a_layer_captured_and_replayed(prism):
    """The layer in two HIP graphs from one pool, replayed in turn with eager work in between: the eager bits every time."""
    inputs = layer_inputs(21)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(prism, *inputs, 2)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, results = [], []
    for k in (2, 3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, pool=graphs[0].pool() if graphs else None):
            results.append(layer(prism, *inputs, k))
        graphs.append(graph)
    for seed in (31, 41, 51):
        for t, fresh in zip(inputs, layer_inputs(seed)):
            t.copy_(fresh)
        for k, graph, result in zip((2, 3), graphs, results):
            eager = [t.clone() for t in (*layer(prism, *inputs, k)[:5], *layer(prism, *inputs, k)[5])]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip((*result[:5], *result[5]), eager):
                assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,experts,k", [(1100, 64, 4), (2900, 64, 4), (5000, 40, 5), (9001, 1024, 3), (4100, 520, 1)])
def test_routes_of_many_tokens_captured(prism, tokens, experts, k):
    """Two graphs, each with its own results and workspaces, replayed in turn with other calls between; every replay against the eager call."""
    logits = [normal(i, tokens, experts).bfloat16() for i in range(4)]
    inputs = [x.clone() for x in logits[:2]]
    for z in logits:
        r = prism.route_topk(z, k)
        want = torch.topk(z.float(), k).values
        assert torch.equal(z.float().gather(1, r.experts.long()), want)
        assert all(torch.equal(a, b) for a, b in zip(r[2:], plain_plan(r.experts, experts)))
    graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, z in zip(graphs, inputs):
        with torch.cuda.graph(g):
            got.append(prism.route_topk(z, k))
    for turn in range(3):
        for i in (0, 1):
            inputs[i].copy_(logits[(turn + i) % 4])
            graphs[i].replay()
        between = prism.route_topk(logits[3], k)
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(got[i], prism.route_topk(logits[(turn + i) % 4], k)))
        assert all(torch.equal(a, b) for a, b in zip(between, prism.route_topk(logits[3], k)))


def test_large_plans_in_graphs_and_on_two_streams(prism):
    """The plan with a workspace: captured, and two at once on two streams."""
    choices = [torch.randint(0, 64, (9000, 4), device=DEV, dtype=torch.int32) for _ in range(2)]
    wants = [plain_plan(c, 64) for c in choices]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, c in zip(streams, choices):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(prism.expert_plan(c, 64))
        torch.cuda.synchronize()
        for g, w in zip(got, wants):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    graph = torch.cuda.CUDAGraph()
    chosen = choices[0].clone()
    with torch.cuda.graph(graph, stream=streams[0]):
        got = prism.expert_plan(chosen, 64)
    for i in (1, 0, 1):
        chosen.copy_(choices[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, wants[i]))


def test_single_tokens_with_weights_in_4_bits(prism):
    """A decoded batch: route, gather, 4-bit products, combine, against the same weights in 64 bits."""
    T, k, E, width, inner, G = 5, 3, 7, 256, 192, 64
    x = normal(1, T, width).bfloat16()
    logits = normal(2, T, E)
    gen = torch.Generator(device=DEV).manual_seed(3)
    q1 = torch.randint(0, 256, (E, inner, width // 2), generator=gen, dtype=torch.uint8, device=DEV)
    s1 = (0.02 * torch.rand(E, inner, width // G, generator=gen, device=DEV)).bfloat16()
    r = prism.route_topk(logits, k)
    y = prism.gemv_w4(prism.expert_gather(x, r.rows, k), q1, s1, G, offsets=r.offsets, out_dtype=torch.float32)
    out = prism.expert_combine(y, r.weights, r.slots)
    w = (torch.stack([q1 & 15, q1 >> 4], -1).reshape(E, inner, width).double() - 8) * s1.double().repeat_interleave(G, 2)
    want = torch.zeros(T, inner, dtype=torch.float64, device=DEV)
    for t in range(T):
        for j in range(k):
            want[t] += float(r.weights[t, j]) * (w[int(r.experts[t, j])] @ x[t].double())
    near(out, want, torch.full_like(want, float(want.abs().max()) * 16), 128 + 24)
