"""Routing and combine against plain definitions, and the layers built on the products."""

import pytest
import torch

from chad_b200 import ops
from chad_b200.attention import scaled_dot_product_attention
from chad_b200.cache import QuantizedKVCache
from chad_b200.experts import QuantizedExperts, QuantizedLinear, quantize_weight
from tests.test_gpu_matmul import check, parts64, reference

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def plain_route(z, k, normalize):
    z = z.cpu().double()
    t, e = z.shape
    key = torch.where(z.isnan(), torch.full_like(z, float("inf")), z)
    # NaN above +inf: a second key breaks that tie, then the index
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    isn = z.isnan().gather(1, order)
    order = order.gather(1, torch.sort((~isn).int(), dim=-1, stable=True).indices)
    experts = order[:, :k]
    mx = z.amax(-1, keepdim=True)
    p = torch.where(z == float("-inf"), torch.zeros_like(z), torch.exp(z - mx))
    chosen = p.gather(1, experts)
    total = (chosen if normalize else p).sum(-1, keepdim=True)
    weights = torch.where(total == 0, torch.zeros_like(chosen), chosen / total)
    flat = experts.flatten()
    perm = torch.sort(flat, stable=True).indices
    slots = torch.empty_like(perm)
    slots[perm] = torch.arange(t * k)
    offsets = torch.zeros(e + 1, dtype=torch.long)
    offsets[1:] = torch.bincount(flat, minlength=e).cumsum(0)
    return experts, weights, perm // k, slots.view(t, k), offsets


def check_route(z, k, normalize):
    got = ops.route_topk(z, k, normalize=normalize)
    want = plain_route(z, k, normalize)
    for name, g, w in zip(got._fields, got, want):
        g = g.cpu()
        if name == "weights":
            # expf (2 ulp), a sum of up to 512 terms over 16 + 5 additions, one divide
            assert torch.equal(g.isnan(), w.isnan())
            ok = (g.double() - w).abs() <= 32 * 2.0 ** -24 * w.abs() + 2.0 ** -126
            assert bool((ok | w.isnan()).all()), name
        else:
            assert g.dtype == torch.int32 and torch.equal(g.long(), w), name


@pytest.mark.parametrize("t,e,k", [
    (t, e, k)
    for e, k in [(1, 1), (7, 3), (32, 8), (60, 4), (128, 8), (200, 16), (512, 10)]
    for t in [0, 1, 5, 63, 64, 65, 200, 1000, 8192, 8193, 20000]
    if t < 2000 or e not in (1, 7, 200)])
def test_route(t, e, k):
    gen = torch.Generator().manual_seed(t * 1009 + e)
    dtype = DT[("bf16", "fp16", "fp32")[(t + e) % 3]]
    z = (torch.randn(t, e, generator=gen) * 2).to(dtype).cuda()  # 16-bit logits hold ties
    for normalize in (True, False):
        check_route(z, k, normalize)


@pytest.mark.parametrize("t,e,k", [(33000, 512, 2), (132000, 200, 3)])
def test_route_of_many_tokens(t, e, k):
    # larger blocks of tokens, whose masks pass 48 KiB of shared memory
    gen = torch.Generator().manual_seed(t)
    check_route(torch.randn(t, e, generator=gen).to(torch.bfloat16).cuda(), k, True)


@pytest.mark.parametrize("t", [6, 90])
def test_route_ties_infinities_and_nan(t):
    z = torch.zeros(t, 40)
    z[1, 5:] = float("-inf")                      # fewer finite logits than choices
    z[2] = float("-inf")                          # nothing left
    z[3, ::2] = -0.0                              # -0 ties with +0
    z[4, 17], z[4, 3] = float("nan"), 2.0
    z[5] = torch.finfo(torch.float32).min
    check_route(z.cuda(), 8, True)
    check_route(z.cuda(), 8, False)
    r = ops.route_topk(z.cuda(), 8)
    assert r.experts[0].tolist() == list(range(8)) and r.experts[3].tolist() == list(range(8))
    assert r.weights[1].tolist()[5:] == [0.0] * 3 and r.weights[2].tolist() == [0.0] * 8
    assert r.experts[4, 0] == 17 and bool(r.weights[4].isnan().all())
    assert bool(r.weights[[0, 1, 2, 3, 5]].isfinite().all())


@pytest.mark.parametrize("e,k", [(40, 3), (128, 8), (512, 16)])
@pytest.mark.parametrize("values", [1, 2, 3, 40])
def test_route_many_equal_logits(e, k, values):
    # from logits that are all the same to about as many of the largest as a warp has lanes
    gen = torch.Generator().manual_seed(e + values)
    z = torch.randint(0, values, (70, e), generator=gen).to(torch.bfloat16)
    check_route(z.cuda(), k, True)
    check_route(z[:9].contiguous().cuda(), k, False)


def test_route_refusals():
    z = torch.zeros(4, 16, device="cuda")
    for bad in (0, 17, -1):
        with pytest.raises(ValueError):
            ops.route_topk(z, bad)
    with pytest.raises(ValueError):
        ops.route_topk(z.t(), 2)
    with pytest.raises(ValueError):
        ops.route_topk(z[0], 2)
    with pytest.raises(TypeError):
        ops.route_topk(z.double(), 2)
    with pytest.raises(RuntimeError):
        ops.route_topk(torch.zeros(4, 600, device="cuda"), 2)


@pytest.mark.parametrize("t,k,n", [(0, 2, 64), (1, 1, 8), (1, 8, 2048), (3, 2, 17), (5, 10, 100),
                                   (130, 4, 1000), (700, 8, 264)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("with_residual", [False, True])
def test_combine(t, k, n, dtype, with_residual):
    gen = torch.Generator().manual_seed(t + 31 * k + n)
    dt = DT[dtype]
    y = torch.randn(max(t * k, 1), n, generator=gen).to(dt).cuda()
    slots = torch.randint(0, y.shape[0], (t, k), generator=gen, dtype=torch.int32).cuda()
    if t > 2:
        slots[0, 0], slots[2, -1] = -1, y.shape[0]  # dropped
    weights = torch.rand(t, k, generator=gen).cuda()
    residual = torch.randn(t, n, generator=gen).to(dt).cuda() if with_residual else None
    got = ops.expert_combine(y, slots, weights, residual=residual)
    held = (slots >= 0) & (slots < y.shape[0])
    terms = y.double()[slots.clamp(0, y.shape[0] - 1).long()] * (weights.double() * held).unsqueeze(-1)
    want, mag = terms.sum(1), terms.abs().sum(1)
    if with_residual:
        want, mag = want + residual.double(), mag + residual.double().abs()
    err = torch.finfo(dt).eps / 2 * want.abs() + (k + 1) * 2.0 ** -23 * mag + torch.finfo(dt).smallest_normal
    check(got, want, err, f"{t}x{k}x{n}")
    if with_residual:  # in place
        assert torch.equal(ops.expert_combine(y, slots, weights, residual=residual, out=residual), got)


def test_combine_refusals():
    y = torch.zeros(8, 32, dtype=torch.bfloat16, device="cuda")
    slots, w = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    with pytest.raises(TypeError):
        ops.expert_combine(y, slots.long(), w)
    with pytest.raises(TypeError):
        ops.expert_combine(y, slots, w.bfloat16())
    with pytest.raises(TypeError):
        ops.expert_combine(y.float(), slots, w)
    with pytest.raises(ValueError):
        ops.expert_combine(y, slots, w[:3])
    with pytest.raises(ValueError):
        ops.expert_combine(y, slots, w, residual=y)
    with pytest.raises(ValueError):
        ops.expert_combine(y[:, ::2], slots, w)


# ---------------------------------------------------------------------------------------
# the layers
# ---------------------------------------------------------------------------------------

def test_quantized_weight_dequantizes_near_the_weight():
    gen = torch.Generator().manual_seed(1)
    w = torch.randn(3, 20, 320, generator=gen).bfloat16().cuda()
    q = quantize_weight(w)
    assert q[0].shape == (3, 20, 40) and q[1].shape == q[2].shape == (3, 20, 5)
    c, s, b = parts64(*q)
    # half a code step, the edge moved by the scale's fit (at most as much again), and the
    # 16-bit roundings of 15 scales and a bias
    err = s.abs() + 2.0 ** -8 * (15 * s.abs() + b.abs())
    assert bool(((c * s + b - w.double()).abs() <= err).all())


@pytest.mark.parametrize("t", [1, 9, 150])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_experts_layer(t, dtype):
    """Route, both grouped products and the combine, each stage against 64 bits on its inputs."""
    gen = torch.Generator().manual_seed(t)
    dt, e, k, f, top = DT[dtype], 10, 192, 128, 3
    layer = QuantizedExperts.from_weights((torch.randn(e, 2 * f, k, generator=gen) * k ** -0.5).to(dt).cuda(),
                                          (torch.randn(e, k, f, generator=gen) * f ** -0.5).to(dt).cuda(), top)
    x = torch.randn(t, k, generator=gen).to(dt).cuda()
    logits = torch.randn(t, e, generator=gen).cuda()
    got = layer(x, logits, residual=x)
    r = ops.route_topk(logits, top)
    want, err = x.double(), torch.zeros(t, k, device="cuda", dtype=torch.double)
    for i in range(t):
        for j in range(top):
            ex = int(r.experts[i, j])
            h, eh = reference(x[i:i + 1], [v[ex] for v in layer.gate_up], "swiglu", dt)
            c, s, b = parts64(*[v[ex] for v in layer.down])
            y = h @ (c * s + b).t()
            _, ey = reference(h.to(dt), [v[ex] for v in layer.down], None, dt)
            p = r.weights[i, j].double()
            want[i] += p * y[0]
            err[i] += p * (ey[0] + (eh @ (c * s + b).abs().t())[0])
    err += torch.finfo(dt).eps / 2 * want.abs() * 1.01 + 2.0 ** -20
    check(got, want, err, f"{t} tokens")


def test_decode_layer_with_attention():
    """Projection, append and attention over the 4-bit cache, output projection: the operators
    as a decode step runs them, captured and replayed, against the same calls made one by one."""
    gen = torch.Generator().manual_seed(3)
    hidden, hq, hkv, d = 256, 8, 2, 64
    dt = torch.bfloat16
    qkv = QuantizedLinear.from_weight((torch.randn((hq + 2 * hkv) * d, hidden, generator=gen) * hidden ** -0.5).to(dt).cuda())
    proj = QuantizedLinear.from_weight((torch.randn(hidden, hq * d, generator=gen) * (hq * d) ** -0.5).to(dt).cuda())
    ffn = QuantizedExperts.from_weights((torch.randn(6, 256, hidden, generator=gen) * hidden ** -0.5).to(dt).cuda(),
                                        (torch.randn(6, hidden, 128, generator=gen) * 128 ** -0.5).to(dt).cuda(), 2)
    router = (torch.randn(hidden, 6, generator=gen) * hidden ** -0.5).to(dt).cuda()

    def step(x, cache):
        p = qkv(x).view(1, 1, hq + 2 * hkv, d).transpose(1, 2)
        q, k, v = p[:, :hq].contiguous(), p[:, hq:hq + hkv].contiguous(), p[:, hq + hkv:].contiguous()
        keys, values = cache.update_and_fetch(k, v)
        a = scaled_dot_product_attention(q, keys, values, cache=cache, scale=d ** -0.5, mask=None)
        h = proj(a.transpose(1, 2).reshape(1, hq * d)) + x
        return ffn(h, h @ router, residual=h)

    cache = QuantizedKVCache(64, 4)
    prompt = torch.randn(1, hkv, 40, d, generator=gen).to(dt).cuda()
    cache.update_and_fetch(prompt, prompt.flip(2))
    x = torch.randn(1, hidden, generator=gen).to(dt).cuda()
    want = step(x, cache)
    assert bool(torch.isfinite(want).all())
    cache.trim(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, cache)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_two_captured_layers_at_once():
    """Two graphs of one layer, replayed on two streams at a time on new data: no workspace is
    shared, and the results are those of calls one by one."""
    gen = torch.Generator().manual_seed(8)
    e, k, f, t = 16, 256, 192, 700
    dt = torch.bfloat16
    layer = QuantizedExperts.from_weights((torch.randn(e, 2 * f, k, generator=gen) * k ** -0.5).to(dt).cuda(),
                                          (torch.randn(e, k, f, generator=gen) * f ** -0.5).to(dt).cuda(), 4)
    xs = [torch.zeros(t, k, dtype=dt, device="cuda") for _ in range(2)]
    zs = [torch.zeros(t, e, device="cuda") for _ in range(2)]
    layer(xs[0], zs[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, z in zip(xs, zs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer(x, z, residual=x))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(3):
        for x, z in zip(xs, zs):
            x.copy_(torch.randn(t, k, generator=gen))
            z.copy_(torch.randn(t, e, generator=gen) * (round_ + 1))
        want = [layer(x, z, residual=x) for x, z in zip(xs, zs)]
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got, w)
