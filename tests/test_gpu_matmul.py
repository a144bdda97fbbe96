"""4-bit products against the definition in 64 bits, at the sizes where they can go wrong."""

import pytest
import torch

from chad_b200 import _lib, ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make_weights(gen, lead, k, dtype):
    """Random codes (every bit pattern) with scales and biases of normal weights."""
    w = torch.randint(-2 ** 31, 2 ** 31, (*lead, k // 8), generator=gen, dtype=torch.int64).int()
    s = (0.004 + 0.004 * torch.rand(*lead, k // 64, generator=gen)).to(dtype)
    s = torch.where(torch.rand(s.shape, generator=gen) < 0.5, s, -s)
    b = (-8 * s.float() * (0.8 + 0.4 * torch.rand(s.shape, generator=gen))).to(dtype)
    return w.cuda(), s.cuda(), b.cuda()


def parts64(w, s, b):
    """Codes, scales and biases of every weight (.., k) in 64 bits."""
    sh = torch.arange(0, 32, 4, device=w.device)
    c = ((w.long().unsqueeze(-1) >> sh) & 15).flatten(-2).double()
    return c, s.double().repeat_interleave(64, -1), b.double().repeat_interleave(64, -1)


def gate(y):
    g, u = y.chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def reference(x, wq, act, dtype):
    """(y, allowed error) of x (m, k) with one weight matrix.

    The kernel for few rows sums codes exactly in products and in fp32 per group: the MMA
    chain of a group is off by at most 4 steps of 2^-22 of its terms' magnitudes (128 + code
    in bf16, which the bias takes off again), the sum over groups by 2^-23 of every partial
    sum. The kernel for many rows rounds a weight once to 16 bits: independent errors of at
    most half a step, a uniform error's deviation over sqrt(3), eight of them allowed. Then
    one rounding of the result; the gated product moves by both factors' errors (|silu'| < 1.1).
    """
    c, s, b = parts64(*wq)
    xd, eps = x.double(), torch.finfo(dtype).eps / 2
    wd = s * c + b
    y = xd @ wd.t()
    k = x.shape[1]
    mag = xd.abs() @ (s.abs() * (128 + c) + (b - 128 * s).abs()).t()
    err = 2.0 ** -20 * mag + (k // 64) * 2.0 ** -23 * (xd.abs() @ wd.abs().t())
    err = err + 8 / 3 ** 0.5 * eps * (xd.square() @ wd.square().t()).sqrt()
    if act:
        g, u = y.chunk(2, -1)
        eg, eu = err.chunk(2, -1)
        silu = g / (1 + torch.exp(-g))
        y, err = silu * u, 1.1 * eg * (u.abs() + eu) + silu.abs() * eu
        err = err + 2.0 ** -21 * y.abs()  # expf and the divide, in fp32
    return y, err + eps * (y.abs() + err) + torch.finfo(dtype).smallest_normal * eps


def check(got, want, err, what):
    off = (got.double() - want).abs()
    worst = (off / err.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert bool((off <= err).all()), f"{what}: {worst:.2f} times the allowed error"


MATMUL = [
    # m, n, k: one value of everything, ragged edges, K chunks of one to four groups and more
    (1, 1, 64), (1, 16, 64), (2, 17, 128), (3, 15, 192), (7, 33, 256), (8, 100, 320),
    (9, 64, 512), (13, 255, 1088), (16, 129, 2048), (17, 40, 576), (31, 257, 704), (64, 300, 1024),
    (65, 128, 256), (130, 200, 320), (257, 96, 832), (300, 513, 64), (1, 5000, 2048),
    (1, 40000, 128), (5, 20001, 320), (40, 9000, 192),
    # more K than any ring of shared-memory stages holds, twice over
    (3, 1000, 4096), (33, 600, 6144), (200, 1300, 4096), (192, 130, 6208),
    # K that leaves shared memory for eight, three, one and no row of x
    (9, 20, 8192), (9, 20, 20480), (3, 20, 65536), (2, 20, 65600),
]


@pytest.mark.parametrize("m,n,k", MATMUL)
@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_matmul(m, n, k, act, dtype):
    gen = torch.Generator().manual_seed(m * 1000003 + n * 1009 + k)
    dt = DT[dtype]
    n += n % 2 if act else 0
    wq = make_weights(gen, (n,), k, dt)
    x = torch.randn(m, k, generator=gen)
    x[:, ::37] *= 8
    x = x.to(dt).cuda()
    got = ops.quantized_matmul(x, wq, activation=act)
    want, err = reference(x, wq, act, dt)
    assert got.shape == want.shape and got.dtype == dt
    check(got, want, err, f"{m}x{n}x{k} {act} {dtype}")


def test_matmul_is_the_same_every_time():
    gen = torch.Generator().manual_seed(4)
    for m in (1, 8, 40, 300):
        wq = make_weights(gen, (520,), 1024, torch.bfloat16)
        x = torch.randn(m, 1024, generator=gen).bfloat16().cuda()
        a = ops.quantized_matmul(x, wq)
        for _ in range(3):
            assert torch.equal(a, ops.quantized_matmul(x, wq))


@pytest.mark.parametrize("m", [1, 12, 90, 300])
def test_rows_of_a_strided_view_and_leading_dims(m):
    gen = torch.Generator().manual_seed(5)
    wq = make_weights(gen, (72,), 192, torch.bfloat16)
    big = torch.randn(m, 640, generator=gen).bfloat16().cuda()
    view = big[:, 64:256]
    want = ops.quantized_matmul(view.contiguous(), wq)
    assert torch.equal(ops.quantized_matmul(view, wq), want)
    lead = view.contiguous().view(m, 1, 192)
    assert torch.equal(ops.quantized_matmul(lead, wq).view(m, 72), want)


@pytest.mark.parametrize("m", [3, 90, 200])
def test_out_is_written_in_place_and_nothing_past_it(m):
    gen = torch.Generator().manual_seed(6)
    wq = make_weights(gen, (75,), 192, torch.float16)
    x = torch.randn(m, 192, generator=gen).half().cuda()
    pool = torch.full((m + 2, 75), 7.0, dtype=torch.float16, device="cuda")
    out = pool[1:m + 1]
    assert ops.quantized_matmul(x, wq, out=out) is out
    assert torch.equal(out, ops.quantized_matmul(x, wq))
    assert bool((pool[0] == 7).all()) and bool((pool[-1] == 7).all())


@pytest.mark.parametrize("m", [4, 70, 200])
def test_a_row_that_is_not_finite_stays_alone(m):
    gen = torch.Generator().manual_seed(7)
    wq = make_weights(gen, (130,), 256, torch.bfloat16)
    x = torch.randn(m, 256, generator=gen).bfloat16().cuda()
    want = ops.quantized_matmul(x, wq)
    x[1, 17] = float("inf")
    x[2, 200] = float("nan")
    got = ops.quantized_matmul(x, wq)
    keep = torch.tensor([i for i in range(m) if i not in (1, 2)], device="cuda")
    assert torch.equal(got[keep], want[keep])
    assert not bool(torch.isfinite(got[1:3]).any())


def test_large_and_small_values():
    """Scales and activations far from 1 keep their relative accuracy."""
    gen = torch.Generator().manual_seed(8)
    for m in (2, 80, 200):
        for ws, xs in ((2.0 ** -20, 2.0 ** 20), (2.0 ** 20, 2.0 ** -20), (2.0 ** -30, 2.0 ** -30)):
            w, s, b = make_weights(gen, (64,), 320, torch.bfloat16)
            s, b = s * ws, b * ws
            x = (torch.randn(m, 320, generator=gen) * xs).bfloat16().cuda()
            got = ops.quantized_matmul(x, (w, s, b))
            want, err = reference(x, (w, s, b), None, torch.bfloat16)
            check(got, want, err, f"m {m} scale {ws} x {xs}")


def test_empty_products():
    gen = torch.Generator().manual_seed(9)
    wq = make_weights(gen, (48,), 128, torch.bfloat16)
    assert ops.quantized_matmul(torch.empty(0, 128, dtype=torch.bfloat16, device="cuda"), wq).shape == (0, 48)


def test_matmul_refuses_what_does_not_fit():
    gen = torch.Generator().manual_seed(10)
    w, s, b = make_weights(gen, (48,), 128, torch.bfloat16)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError):
        ops.quantized_matmul(x.half(), (w, s, b))
    with pytest.raises(TypeError):
        ops.quantized_matmul(x.float(), (w, s.float(), b.float()))
    with pytest.raises(TypeError):
        ops.quantized_matmul(x, (w.float(), s, b))
    with pytest.raises(ValueError):
        ops.quantized_matmul(x[:, :64], (w, s, b))
    with pytest.raises(ValueError):
        ops.quantized_matmul(x, (w, s[:, :1].contiguous(), b))
    with pytest.raises(ValueError):
        ops.quantized_matmul(x, (w, s, b[:24]))
    with pytest.raises(ValueError):
        ops.quantized_matmul(x, (w[::2], s[::2], b[::2]))
    with pytest.raises(ValueError):
        ops.quantized_matmul(x, (w, s, b), activation="gelu")
    with pytest.raises(ValueError):
        ops.quantized_matmul(x, (w, s, b), out=torch.empty(2, 47, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        ops.quantized_matmul(x.t().contiguous().t(), (w, s, b))
    with pytest.raises(_lib.QKVError):
        ops.quantized_matmul(x, (w[:47], s[:47], b[:47]), activation="swiglu")
    with pytest.raises(_lib.QKVError):  # 8-bit codes of K = 64
        ops.quantized_matmul(x[:, :64].contiguous(), (w, s[:, :1].contiguous(), b[:, :1].contiguous()), bits=8)


# ---------------------------------------------------------------------------------------
# grouped
# ---------------------------------------------------------------------------------------

GROUPED = [
    # rows per expert, n, k
    ([1], 16, 64), ([0, 3, 0, 1], 40, 128), ([1, 1, 1, 1, 1, 1, 1, 1], 65, 256),
    ([9, 0, 8, 7, 25], 100, 320), ([0, 0, 0, 5], 33, 192), ([200, 1, 0, 3], 72, 256),
    ([2] * 70, 48, 128), ([40, 50, 60, 70, 0, 80], 130, 512), ([300, 20], 257, 448),
    ([129, 256, 127], 128, 1024), ([64] * 4, 512, 64), ([17] * 33, 144, 1088),
]


@pytest.mark.parametrize("counts,n,k", GROUPED)
@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped(counts, n, k, act, dtype, gather):
    e, r = len(counts), sum(counts)
    gen = torch.Generator().manual_seed(r * 1009 + n * 13 + k)
    dt = DT[dtype]
    n += n % 2 if act else 0
    wq = make_weights(gen, (e, n), k, dt)
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    if gather:  # repeated rows, as tokens with several experts
        x = torch.randn(max(1, r // 2), k, generator=gen).to(dt).cuda()
        rows = torch.randint(0, x.shape[0], (r,), generator=gen, dtype=torch.int32).cuda()
        src = x[rows.long()]
    else:
        x = src = torch.randn(r, k, generator=gen).to(dt).cuda()
        rows = None
    got = ops.grouped_quantized_matmul(x, wq, offsets, rows=rows, activation=act)
    at = 0
    for i, c in enumerate(counts):
        if c:
            want, err = reference(src[at:at + c], [t[i] for t in wq], act, dt)
            check(got[at:at + c], want, err, f"expert {i} of {counts} {n}x{k} {act} {dtype}")
        at += c


@pytest.mark.parametrize("counts", [[1, 0, 2] * 100, [0] * 699 + [11], [21, 0, 0, 9] * 275,
                                    [3] * 1025, [40, 0, 0, 0] * 260])
def test_more_experts_than_threads(counts):
    # more than a block has threads, and more than the kernel for many rows takes
    gen = torch.Generator().manual_seed(len(counts))
    wq = make_weights(gen, (len(counts), 24), 128, torch.bfloat16)
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    x = torch.randn(sum(counts), 128, generator=gen).bfloat16().cuda()
    got = ops.grouped_quantized_matmul(x, wq, offsets)
    at = 0
    for i, c in enumerate(counts):
        if c:
            want, err = reference(x[at:at + c], [t[i] for t in wq], None, torch.bfloat16)
            check(got[at:at + c], want, err, f"expert {i} of {len(counts)}")
        at += c


@pytest.mark.parametrize("m,n", [(8193, 1), (65528, 3), (65529, 3), (70000, 16), (600000, 1)])
def test_many_rows_through_few_weights(m, n):
    gen = torch.Generator().manual_seed(m)
    wq = make_weights(gen, (n,), 64, torch.float16)
    x = torch.randn(m, 64, generator=gen).half().cuda()
    want, err = reference(x, wq, None, torch.float16)
    check(ops.quantized_matmul(x, wq), want, err, f"{m} rows, {n} weights")


@pytest.mark.parametrize("counts", [[3, 0, 5], [90, 0, 100]])
def test_rows_outside_the_offsets_are_left_alone(counts):
    gen = torch.Generator().manual_seed(11)
    wq = make_weights(gen, (3, 50), 128, torch.bfloat16)
    r = sum(counts) + 7
    x = torch.randn(r, 128, generator=gen).bfloat16().cuda()
    off = torch.tensor([2, 2 + counts[0], 2 + counts[0], 2 + sum(counts)], dtype=torch.int32, device="cuda")
    out = torch.full((r, 50), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.grouped_quantized_matmul(x, wq, off, out=out)
    assert bool((out[:2] == 9).all()) and bool((out[2 + sum(counts):] == 9).all())
    for i in (0, 2):
        a, b = int(off[i]), int(off[i + 1])
        want, err = reference(x[a:b], [t[i] for t in wq], None, torch.bfloat16)
        check(out[a:b], want, err, f"expert {i}")


@pytest.mark.parametrize("per", [3, 120])
def test_bad_indices_stay_inside(per):
    """Rows outside x read zeros; offsets outside [0, R] are clamped; a decreasing pair is empty."""
    gen = torch.Generator().manual_seed(12)
    wq = make_weights(gen, (3, 40), 128, torch.bfloat16)
    r = 2 * per
    x = torch.randn(r, 128, generator=gen).bfloat16().cuda()
    rows = torch.arange(r, dtype=torch.int32)
    rows[1], rows[per] = -1, r
    off = torch.tensor([-5, per, per - 2, 2 ** 31 - 1], dtype=torch.int32)
    off[2] = per
    out = ops.grouped_quantized_matmul(x, wq, off.cuda(), rows=rows.cuda())
    src = x.clone()
    src[1] = src[per] = 0
    for i, (a, b) in ((0, (0, per)), (2, (per, r))):
        want, err = reference(src[a:b], [t[i] for t in wq], None, torch.bfloat16)
        check(out[a:b], want, err, f"expert {i}")
    assert bool((out[1] == 0).all()) and bool((out[per] == 0).all())
    # decreasing: the second expert is empty and the third starts earlier again
    out = torch.full((r, 40), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.grouped_quantized_matmul(x, wq, torch.tensor([per, 1, 1, 1], dtype=torch.int32, device="cuda"), out=out)
    assert bool((out == 9).all())


def test_grouped_of_no_rows():
    gen = torch.Generator().manual_seed(13)
    wq = make_weights(gen, (3, 40), 128, torch.bfloat16)
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 128, dtype=torch.bfloat16, device="cuda")
    assert ops.grouped_quantized_matmul(x, wq, off).shape == (0, 40)
    out = torch.full((5, 40), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.grouped_quantized_matmul(torch.zeros(5, 128, dtype=torch.bfloat16, device="cuda"), wq, off, out=out)
    assert bool((out == 9).all())


def test_grouped_refuses_what_does_not_fit():
    gen = torch.Generator().manual_seed(14)
    wq = make_weights(gen, (3, 40), 128, torch.bfloat16)
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda")
    off = torch.tensor([0, 1, 2, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError):
        ops.grouped_quantized_matmul(x, wq, off.long())
    with pytest.raises(TypeError):
        ops.grouped_quantized_matmul(x, wq, off, rows=torch.zeros(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ops.grouped_quantized_matmul(x, wq, off[:3].contiguous())
    with pytest.raises(ValueError):
        ops.grouped_quantized_matmul(x, [t[0] for t in wq], off)
    with pytest.raises(ValueError):
        ops.grouped_quantized_matmul(x[None], wq, off)
    with pytest.raises(ValueError):
        ops.grouped_quantized_matmul(x, wq, off, rows=torch.zeros(2, 2, dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------------------------------
# streams, graphs, offsets past 32 bits
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [1, 40, 300])
def test_two_streams_at_once(m):
    gen = torch.Generator().manual_seed(15)
    wq = make_weights(gen, (640,), 1024, torch.bfloat16)
    xs = [torch.randn(m, 1024, generator=gen).bfloat16().cuda() for _ in range(2)]
    want = [ops.quantized_matmul(x, wq, activation="swiglu") for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.quantized_matmul(xs[i], wq, activation="swiglu"))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(v, want[i]) for v in got[i])


@pytest.mark.parametrize("m", [1, 40, 300])
def test_captured_and_replayed_on_new_data(m):
    gen = torch.Generator().manual_seed(16)
    wq = make_weights(gen, (4, 96), 512, torch.bfloat16)
    one = tuple(t[0] for t in wq)
    x = torch.randn(m, 512, generator=gen).bfloat16().cuda()
    off = torch.zeros(5, dtype=torch.int32, device="cuda")
    off[1:] = m
    out = torch.zeros(m, 96, dtype=torch.bfloat16, device="cuda")
    ops.quantized_matmul(x, one, activation="swiglu")
    ops.grouped_quantized_matmul(x, wq, off, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = ops.quantized_matmul(x, one, activation="swiglu")
        ops.grouped_quantized_matmul(x, wq, off, out=out)
    for seed in range(3):
        x.copy_(torch.randn(m, 512, generator=gen).bfloat16())
        off[1:4] = m * seed // 3
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ops.quantized_matmul(x, one, activation="swiglu"))
        assert torch.equal(out, ops.grouped_quantized_matmul(x, wq, off))


def test_weights_past_32_bit_offsets():
    """Stacked experts of more than 2^32 values: the last expert's rows are found."""
    e, n, k = 70, 16384, 4096
    assert e * n * k > 2 ** 32
    w = torch.zeros(e, n, k // 8, dtype=torch.int32, device="cuda")
    s = torch.zeros(e, n, k // 64, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(17)
    lw, ls, lb = make_weights(gen, (n,), k, torch.bfloat16)
    w[-1], s[-1] = lw, ls
    b = torch.zeros_like(s)
    b[-1] = lb
    for r in (3, 200):
        x = torch.randn(r, k, generator=gen).bfloat16().cuda()
        off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
        off[-1] = r
        got = ops.grouped_quantized_matmul(x, (w, s, b), off)
        want, err = reference(x, (lw, ls, lb), None, torch.bfloat16)
        check(got, want, err, f"last of {e} experts, {r} rows")


# ---------------------------------------------------------------------------------------
# the kernel for many rows, at sizes that are sure to reach it
# ---------------------------------------------------------------------------------------

def takes_many(r, e, n, k):
    """Does the library take these rows to the kernel that gathers into a workspace?"""
    return _lib.load().qkv_matmul_workspace_size(r, e, n, k, 1) > 0


@pytest.mark.parametrize("m,n,k", [
    (300, 1000, 1088), (1000, 514, 832), (2000, 302, 320), (4000, 600, 64), (5000, 258, 128),
    (9000, 34, 2112), (193, 2000, 704), (33, 20000, 960), (17, 40002, 1984), (200, 1301, 4096),
    (384, 900, 1984), (64, 8190, 1024), (1537, 1026, 576), (100, 16384, 192),
])
@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_matmul_of_many_rows(m, n, k, act, dtype):
    n += n % 2 if act else 0
    assert takes_many(m, 1, n, k)
    gen = torch.Generator().manual_seed(m * 7 + n)
    dt = DT[dtype]
    wq = make_weights(gen, (n,), k, dt)
    x = torch.randn(m, k, generator=gen).to(dt).cuda()
    want, err = reference(x, wq, act, dt)
    got = ops.quantized_matmul(x, wq, activation=act)
    check(got, want, err, f"{m} x {k} through {n} {act} {dtype}")
    # a strided view, results in place and nothing past them, the same once more
    big = torch.randn(m, k + 72, generator=gen).to(dt).cuda()
    big[:, 40:40 + k] = x
    pool = torch.full((m + 2, got.shape[1]), 7.0, dtype=dt, device="cuda")
    ops.quantized_matmul(big[:, 40:40 + k], wq, activation=act, out=pool[1:m + 1])
    assert torch.equal(pool[1:m + 1], got)
    assert bool((pool[0] == 7).all()) and bool((pool[-1] == 7).all())


@pytest.mark.parametrize("counts,n,k", [
    ([200, 1, 0, 300, 17], 700, 1088), ([129, 256, 127], 640, 1024), ([64] * 8, 1100, 704),
    ([500, 0, 0, 1], 702, 960), ([17] * 33, 1026, 320), ([2] * 10 + [900], 500, 576),
    ([0, 0, 1000], 514, 512), ([193, 385, 31, 33, 0, 16, 15], 900, 640),
    ([3, 90, 0, 40, 250, 8, 1, 1, 60, 11], 4098, 192), ([70] * 60, 130, 1408),
])
@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_of_many_rows(counts, n, k, act, dtype, gather):
    assert takes_many(sum(counts), len(counts), n, k)
    test_grouped(counts, n, k, act, dtype, gather)


def test_many_rows_that_are_not_finite_or_not_there():
    gen = torch.Generator().manual_seed(18)
    r, n, k = 640, 900, 640
    assert takes_many(r, 3, n, k) and takes_many(r, 1, n, k)
    wq = make_weights(gen, (3, n), k, torch.bfloat16)
    one = tuple(t[0] for t in wq)
    x = torch.randn(r, k, generator=gen).bfloat16().cuda()
    want = ops.quantized_matmul(x, one)
    y = x.clone()
    y[1, 17], y[200, 600] = float("inf"), float("nan")
    got = ops.quantized_matmul(y, one)
    keep = torch.tensor([i for i in range(r) if i not in (1, 200)], device="cuda")
    assert torch.equal(got[keep], want[keep])
    assert not bool(torch.isfinite(got[[1, 200]]).any())
    # rows before, between and after the experts' are left alone
    off = torch.tensor([2, 250, 250, 600], dtype=torch.int32, device="cuda")
    out = torch.full((r, n), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.grouped_quantized_matmul(x, wq, off, out=out)
    assert bool((out[:2] == 9).all()) and bool((out[600:] == 9).all())
    for i, (a, b) in ((0, (2, 250)), (2, (250, 600))):
        ref, err = reference(x[a:b], [t[i] for t in wq], None, torch.bfloat16)
        check(out[a:b], ref, err, f"expert {i}")
    # bad offsets and rows stay inside
    rows = torch.arange(r, dtype=torch.int32)
    rows[1], rows[300] = -1, r
    off = torch.tensor([-5, 320, 320, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    out = ops.grouped_quantized_matmul(x, wq, off, rows=rows.cuda())
    src = x.clone()
    src[1] = src[300] = 0
    for i, (a, b) in ((0, (0, 320)), (2, (320, r))):
        ref, err = reference(src[a:b], [t[i] for t in wq], None, torch.bfloat16)
        check(out[a:b], ref, err, f"expert {i}")
    out = torch.full((r, n), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.grouped_quantized_matmul(x, wq, torch.tensor([r, 1, 1, 1], dtype=torch.int32, device="cuda"), out=out)
    assert bool((out == 9).all())


def test_many_rows_on_two_streams_and_in_graphs():
    gen = torch.Generator().manual_seed(19)
    r, e, n, k = 700, 4, 1000, 512
    assert takes_many(r, e, n, k) and takes_many(r, 1, n, k)
    wq = make_weights(gen, (e, n), k, torch.bfloat16)
    one = tuple(t[0] for t in wq)
    xs = [torch.randn(r, k, generator=gen).bfloat16().cuda() for _ in range(2)]
    rows = torch.randint(0, r, (r,), generator=gen, dtype=torch.int32).cuda()
    off = torch.tensor([0, 100, 100, 333, r], dtype=torch.int32, device="cuda")

    def calls(x):
        return (ops.quantized_matmul(x, one, activation="swiglu"),
                ops.grouped_quantized_matmul(x, wq, off, rows=rows))

    want = [calls(x) for x in xs]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(calls(x))
        graphs.append(graph)
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(calls(xs[i]))
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        for pair in (*got[i], outs[i]):
            assert torch.equal(pair[0], want[i][0]) and torch.equal(pair[1], want[i][1])
    # new data; the pair 200, 100 decreases, and rows 100 to 199 are the first and third expert's
    xs[0].copy_(xs[1])
    off[1] = 200
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], calls(xs[0])[0])
    by = [ops.quantized_matmul(xs[0][rows.long()], tuple(t[i] for t in wq)) for i in (0, 2, 3)]
    got = outs[0][1]
    assert torch.equal(got[:100], by[0][:100])
    assert bool(((got == by[0]) | (got == by[1]))[100:200].all())
    assert torch.equal(got[200:333], by[1][200:333]) and torch.equal(got[333:], by[2][333:])
