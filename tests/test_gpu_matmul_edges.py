"""4-bit products where several calls, kernels or experts meet."""

import pytest
import torch

from chad_b200 import ops
from tests.test_gpu_matmul import check, gate, make_weights, parts64, reference, takes_many

pytestmark = pytest.mark.gpu


# ascending pairs that together have more rows than x, with pairs that decrease between them
OVERLAPPING = [[0, 50, 0, 50, 0, 50, 100], [40, 100, 0, 100], [0, 100] * 6 + [90, 100],
               [0, 64, 0, 64, 0, 64, 0, 64, 0, 64, 0, 64, 100]]


@pytest.mark.parametrize("offsets", OVERLAPPING)
@pytest.mark.parametrize("empty", [0, 300])
def test_rows_of_experts_that_overlap(offsets, empty):
    """A row of one expert has its result, every value of a row of several that of one of them."""
    gen = torch.Generator().manual_seed(sum(offsets))
    offsets = offsets[:1] * empty + offsets
    e, r = len(offsets) - 1, max(offsets)
    wq = make_weights(gen, (e, 24), 128, torch.bfloat16)
    x = torch.randn(r, 128, generator=gen).bfloat16().cuda()
    out = torch.full((r, 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.grouped_quantized_matmul(x, wq, torch.tensor(offsets, dtype=torch.int32, device="cuda"), out=out)
    held = torch.zeros(r, dtype=torch.bool, device="cuda")
    right = torch.zeros(r, 24, dtype=torch.bool, device="cuda")
    for i, (a, b) in enumerate(zip(offsets, offsets[1:])):
        if a < b:
            want, err = reference(x[a:b], [t[i] for t in wq], None, torch.bfloat16)
            right[a:b] |= ((out[a:b].double() - want).abs() <= err)
            held[a:b] = True
    assert torch.equal(right, held[:, None].expand_as(right)) and bool(out[~held].isnan().all())


@pytest.mark.parametrize("m", [1, 4000])
def test_gates_far_below_zero(m):
    """silu of -80 to -88 times a large up projection: about 2^-126 times 2^70, not zero.

    One-hot rows and weights of whole steps, so that gate and up are exact; the largest argument of
    expf is 88, inside its range, and 2^-21 covers it, the divide and two products as in `reference`.
    """
    n, k, dt = 1024, 128, torch.bfloat16
    assert takes_many(m, 1, n, k) == (m > 1)
    half = n // 2
    w = torch.zeros(n, k // 8, dtype=torch.int32, device="cuda")  # every weight is its bias
    s = torch.ones(n, k // 64, dtype=dt, device="cuda")
    b = torch.empty(n, k // 64, dtype=dt, device="cuda")
    b[:half] = -80 - 0.5 * (torch.arange(half, device="cuda") % 17).to(dt)[:, None]
    b[half:] = 2.0 ** 70
    x = torch.zeros(m, k, dtype=dt, device="cuda")
    x[torch.arange(m), torch.arange(m) % k] = 1
    got = ops.quantized_matmul(x, (w, s, b), activation="swiglu").double()
    gate = b[:half, 0].double()
    want = (gate / (1 + torch.exp(-gate)) * 2.0 ** 70).expand(m, half)
    assert bool((gate == -88).any())
    assert bool(((got - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs()).all())


@pytest.mark.parametrize("m,k", [(1, 67392), (2, 67392), (1, 67456), (9, 14336), (5, 28672)])
def test_longest_rows_beside_the_weights_stages(m, k):
    gen = torch.Generator().manual_seed(k + m)
    wq = make_weights(gen, (40,), k, torch.bfloat16)
    x = torch.randn(m, k, generator=gen).bfloat16().cuda()
    want, err = reference(x, wq, None, torch.bfloat16)
    check(ops.quantized_matmul(x, wq), want, err, f"{m} rows of {k}")


@pytest.mark.parametrize("k", [14336, 28672, 67392])
def test_experts_with_fewer_rows_to_a_pass(k):
    gen = torch.Generator().manual_seed(k)
    counts = [3, 0, 7, 1, 2]
    wq = make_weights(gen, (5, 24), k, torch.bfloat16)
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    x = torch.randn(sum(counts), k, generator=gen).bfloat16().cuda()
    got = ops.grouped_quantized_matmul(x, wq, offsets)
    for i, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        if a < b:
            want, err = reference(x[a:b], [t[i] for t in wq], None, torch.bfloat16)
            check(got[a:b], want, err, f"expert {i}")


def reference_of_few_rows(x, wq, act, dtype):
    """(y, allowed error) where no weight is rounded: the terms of `reference` but for that one.

    Also y of weights rounded to dtype, from the oracle, which the bound can tell apart up to a K of
    about 2048 (past that the sums' own terms are larger).
    """
    c, s, b = parts64(*wq)
    xd, wd, eps = x.double(), s * c + b, torch.finfo(dtype).eps / 2
    y, rounded = xd @ wd.t(), xd @ wd.to(dtype).double().t()
    zero = 128 if dtype is torch.bfloat16 else 0  # a code enters the MMA as zero + code
    mag = xd.abs() @ (s.abs() * (zero + c) + (b - zero * s).abs()).t()
    err = 2.0 ** -20 * mag + (x.shape[1] // 64) * 2.0 ** -23 * (xd.abs() @ wd.abs().t())
    if act:
        g, u = y.chunk(2, -1)
        eg, eu = err.chunk(2, -1)
        silu = g / (1 + torch.exp(-g))
        y, err = silu * u, 1.1 * eg * (u.abs() + eu) + silu.abs() * eu
        err = err + 2.0 ** -21 * y.abs()
        rounded = gate(rounded)
    return y, err + eps * (y.abs() + err) + torch.finfo(dtype).smallest_normal * eps, rounded


@pytest.mark.parametrize("m,n,k", [(1, 300, 64), (1, 515, 2048), (3, 1000, 4096), (8, 260, 1088), (16, 130, 2048),
                                   (40, 100, 192), (48, 90, 4096), (2, 60, 20480)])
@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_rows_round_no_weight(m, n, k, act, dtype):
    n += n % 2 if act else 0
    assert not takes_many(m, 1, n, k)
    gen = torch.Generator().manual_seed(m + n + k)
    wq = make_weights(gen, (n,), k, dtype)
    x = torch.randn(m, k, generator=gen).to(dtype).cuda()
    want, err, rounded = reference_of_few_rows(x, wq, act, dtype)
    assert k > 2048 or bool(((rounded - want).abs() > err).any())
    check(ops.quantized_matmul(x, wq, activation=act), want, err, f"{m}x{n}x{k}")


@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_rows_of_experts_round_no_weight(act, dtype):
    gen = torch.Generator().manual_seed(21)
    counts, n, k = [3, 0, 9, 1, 8], 200, 1088
    assert not takes_many(sum(counts), len(counts), n, k)
    wq = make_weights(gen, (len(counts), n), k, dtype)
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    x = torch.randn(sum(counts), k, generator=gen).to(dtype).cuda()
    got = ops.grouped_quantized_matmul(x, wq, offsets, activation=act)
    for i, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        if a < b:
            want, err, _ = reference_of_few_rows(x[a:b], [t[i] for t in wq], act, dtype)
            check(got[a:b], want, err, f"expert {i}")


@pytest.mark.parametrize("m", [1, 9, 2000])
@pytest.mark.parametrize("k", [192, 512, 1024])
def test_scales_that_begin_anywhere(m, k):
    """Scales and biases from an odd place of a larger tensor, for every way that they are copied."""
    gen = torch.Generator().manual_seed(m + k)
    n = 1000
    assert takes_many(m, 1, n, k) == (m == 2000)
    w, s, b = make_weights(gen, (n,), k, torch.bfloat16)
    x = torch.randn(m, k, generator=gen).bfloat16().cuda()
    want = ops.quantized_matmul(x, (w, s, b))
    for off_s, off_b in ((1, 1), (2, 4), (4, 0), (8, 3)):
        views = []
        for t, off in ((s, off_s), (b, off_b)):
            pool = torch.full((t.numel() + 16,), float("nan"), dtype=t.dtype, device="cuda")
            views.append(pool[off:off + t.numel()].view(t.shape).copy_(t))
        assert torch.equal(ops.quantized_matmul(x, (w, *views)), want)
