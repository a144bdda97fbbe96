"""The projections and expert layers around the attention: what is measured of them.

Four operators, over weights in the affine 4-bit format of the cache (codes packed LSB-first
in 32-bit words, a scale and a bias per group of 64 along the contraction):

  matmul   x W^T for one weight matrix, from one token to a prefill chunk; with "swiglu" the
           weight's first half of rows are the gate, the second half the up projection, and
           silu(gate) * up comes back
  grouped  the same with one weight matrix per expert over rows sorted by expert
  route    the k largest logits per token, their softmax weights, and the stable order of
           the (token, expert) pairs by expert
  combine  the weighted sum of every token's expert rows, with an optional residual

`own` false computes them from elementary torch operations in 32 bits, rounded once at the
end; `own` true calls the package.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 64


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def listed():
    return [
        # one decode token through the fused q/k/v projection of 32 query and 4 key/value
        # heads of 128: a small matrix, where the launch counts
        {"name": "matvec-qkv", "op": "matmul", "m": 1, "n": 5120, "k": 2048, "act": "", "dtype": "bf16"},
        # one decode token through the output head of an odd-sized vocabulary: pure bandwidth
        {"name": "matvec-head", "op": "matmul", "m": 1, "n": 131071, "k": 2048, "act": "", "dtype": "fp16"},
        # an 8-token verify block through a gated feed-forward's first projection
        {"name": "verify-mlp", "op": "matmul", "m": 8, "n": 12288, "k": 2048, "act": "swiglu", "dtype": "bf16"},
        # a decode batch of 48 sequences through the attention's output projection
        {"name": "batch-out", "op": "matmul", "m": 48, "n": 2048, "k": 4096, "act": "", "dtype": "bf16"},
        # a 2048-token prefill chunk through the q/k/v projection: matrix-pipe bound
        {"name": "prefill-qkv", "op": "matmul", "m": 2048, "n": 5120, "k": 2048, "act": "", "dtype": "bf16"},
        # one decode token through the gate/up projections of its 8 experts of 128
        {"name": "experts-token", "op": "grouped", "t": 1, "top": 8, "e": 128, "n": 1536, "k": 2048, "act": "swiglu",
         "gather": True, "skew": 0.0, "dtype": "bf16"},
        # a ragged batch with popular experts through the down projection (rows in order)
        {"name": "experts-skewed", "op": "grouped", "t": 333, "top": 4, "e": 60, "n": 2048, "k": 1408, "act": "",
         "gather": False, "skew": 1.0, "dtype": "fp16"},
        # a 2048-token prefill chunk through the gate/up projections of 128 experts
        {"name": "experts-prefill", "op": "grouped", "t": 2048, "top": 8, "e": 128, "n": 1536, "k": 2048, "act": "swiglu",
         "gather": True, "skew": 0.3, "dtype": "bf16"},
        # routing of a decode batch, and of a long prefill chunk
        {"name": "route-decode", "op": "route", "t": 16, "top": 8, "e": 128, "normalize": True, "dtype": "bf16"},
        {"name": "route-prefill", "op": "route", "t": 8192, "top": 8, "e": 256, "normalize": True, "dtype": "fp32"},
        # the experts' rows back into token order: one token, and a prefill chunk
        {"name": "combine-token", "op": "combine", "t": 1, "top": 8, "n": 2048, "residual": True, "dtype": "bf16"},
        {"name": "combine-prefill", "op": "combine", "t": 2048, "top": 8, "n": 2048, "residual": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    top_flops = work(listed()[7])["flops"]
    top_bytes = work(listed()[1])["bytes"] * 2
    while True:
        op = rng.choice(["matmul", "matmul", "matmul", "grouped", "grouped", "grouped", "route", "combine"])
        dtype = rng.choice(["bf16", "fp16"])
        if op == "matmul":
            act = rng.choice(["", "", "swiglu"])
            n = _log(rng, 16, 131072)
            c = {"op": op, "m": rng.choice([_log(rng, 1, 16), _log(rng, 1, 256), _log(rng, 1, 4096)]), "n": n + n % 2 if act else n,
                 "k": 64 * _log(rng, 1, 96), "act": act, "dtype": dtype}
        elif op == "grouped":
            e = _log(rng, 2, 256)
            act = rng.choice(["", "swiglu"])
            n = _log(rng, 16, 4096)
            c = {"op": op, "t": _log(rng, 1, 4096), "top": min(e, rng.randint(1, 10)), "e": e, "n": n + n % 2 if act else n,
                 "k": 64 * _log(rng, 1, 64), "act": act, "gather": rng.random() < 0.5, "skew": rng.choice([0.0, 0.3, 1.0]), "dtype": dtype}
        elif op == "route":
            e = _log(rng, 2, 512)
            c = {"op": op, "t": _log(rng, 1, 16384), "top": min(e, rng.randint(1, 10)), "e": e, "normalize": rng.random() < 0.7,
                 "dtype": rng.choice(["bf16", "fp16", "fp32"])}
        else:
            c = {"op": op, "t": _log(rng, 1, 8192), "top": rng.randint(1, 10), "n": _log(rng, 16, 8192), "residual": rng.random() < 0.5,
                 "dtype": dtype}
        w = work(c)
        if w["flops"] <= top_flops and w["bytes"] <= top_bytes:
            return c


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "fp32" else 2
    if op == "route":
        t, k, e = case["t"], case["top"], case["e"]
        # logits once; expert, weight, row and slot of every pair; the offsets
        return {"bytes": t * e * size + t * k * 16 + (e + 1) * 4, "flops": t * e * 2}
    if op == "combine":
        t, k, n = case["t"], case["top"], case["n"]
        return {"bytes": (t * k + t * (2 if case["residual"] else 1)) * n * size + t * k * 8, "flops": 2 * t * k * n}
    n, k = case["n"], case["k"]
    out = n // 2 if case["act"] else n
    weights = n * (k // 2 + k // GROUP * 2 * size)
    if op == "matmul":
        m = case["m"]
        return {"bytes": weights + m * (k + out) * size, "flops": 2 * m * n * k}
    t, r, e = case["t"], case["t"] * case["top"], case["e"]
    # a token's experts are distinct; over many tokens nearly all experts have rows
    used = e * (1 - (1 - case["top"] / e) ** t)
    rows_in = t if case["gather"] else r
    return {"bytes": used * weights + (rows_in * k + r * out) * size + r * 4, "flops": 2 * r * n * k}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _weights(gen, rows, k, dtype, spread):
    """Normal weights in the affine 4-bit format: (w int32 (rows, k/8), scales, biases)."""
    # a few thousand million values at most: quantized in slices to bound the memory
    w, s, b = [], [], []
    step = max(1, (1 << 27) // k)
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int64)
    for at in range(0, rows, step):
        v = torch.randn(min(step, rows - at), k // GROUP, GROUP, device="cuda", generator=gen) * spread
        mx, mn = v.amax(-1, keepdim=True), v.amin(-1, keepdim=True)
        side = mn.abs() > mx.abs()
        scale = ((mx - mn) / 15).clamp_min(1e-7)
        scale = torch.where(side, scale, -scale)
        edge = torch.where(side, mn, mx)
        q0 = (edge / scale).round()
        scale = torch.where(q0 != 0, edge / q0, scale)
        bias = torch.where(q0 != 0, edge, torch.zeros_like(edge))
        c = ((v - bias) / scale).round().clamp(0, 15).to(torch.int32).view(v.shape[0], k // 8, 8)
        word = c[..., 0].clone()
        for i in range(1, 8):
            word |= c[..., i] << int(shifts[i])
        w.append(word)
        s.append(scale.squeeze(-1).to(dtype))
        b.append(bias.squeeze(-1).to(dtype))
    return torch.cat(w), torch.cat(s), torch.cat(b)


def _tokens(gen, t, k, dtype):
    """Normalised activations with a few outlier channels, as after a norm layer."""
    x = torch.randn(t, k, device="cuda", generator=gen)
    x[:, torch.tensor([3, 37, 50, 61], device="cuda")] *= 8
    return x.to(dtype)


def _routing(gen, t, top, e, skew):
    """Sorted routing of t tokens: token of every sorted row, offsets by expert, slots."""
    logits = torch.randn(t, e, device="cuda", generator=gen) + skew * torch.randn(e, device="cuda", generator=gen)
    experts = logits.topk(top, dim=-1).indices
    order = torch.sort(experts.flatten(), stable=True).indices
    counts = torch.bincount(experts.flatten(), minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return (order // top).to(torch.int32), offsets, int(counts.max())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "route":
        # logits of a router: normal, with popular experts
        z = torch.randn(case["t"], case["e"], device="cuda", generator=gen) + 0.5 * torch.randn(case["e"], device="cuda", generator=gen)
        s["logits"] = z.to(dtype)
    elif op == "combine":
        t, k, n = case["t"], case["top"], case["n"]
        s["y"] = torch.randn(t * k, n, device="cuda", generator=gen).to(dtype)
        s["slots"] = torch.randperm(t * k, device="cuda", generator=gen).view(t, k).to(torch.int32)
        s["weights"] = torch.rand(t, k, device="cuda", generator=gen).softmax(-1)
        s["residual"] = torch.randn(t, n, device="cuda", generator=gen).to(dtype) if case["residual"] else None
    elif op == "matmul":
        s["x"] = _tokens(gen, case["m"], case["k"], dtype)
        s["w"] = _weights(gen, case["n"], case["k"], dtype, case["k"] ** -0.5)
    else:
        t, e, n, k = case["t"], case["e"], case["n"], case["k"]
        rows, s["offsets"], s["most"] = _routing(gen, t, case["top"], e, case["skew"])
        s["rows"] = rows if case["gather"] else None
        s["x"] = _tokens(gen, t if case["gather"] else t * case["top"], k, dtype)
        s["w"] = tuple(v.view(e, n, -1) for v in _weights(gen, e * n, k, dtype, k ** -0.5))
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def _dequantize(w):
    """(..., k) float32 values of 4-bit codes: scale * code + bias."""
    word, scale, bias = w
    shifts = torch.arange(0, 32, 4, device=word.device, dtype=torch.int32)
    codes = (word.unsqueeze(-1) >> shifts) & 15
    codes = codes.view(*scale.shape, GROUP).float()
    return (codes * scale.float().unsqueeze(-1) + bias.float().unsqueeze(-1)).flatten(-2)


def _activate(y, act):
    if not act:
        return y
    gate, up = y.chunk(2, dim=-1)
    return gate / (1 + torch.exp(-gate)) * up


def _plain_matmul(s):
    y = s["x"].float() @ _dequantize(s["w"]).t()
    return _activate(y, s["case"]["act"]).to(s["x"].dtype)


def _plain_grouped(s):
    # every expert's rows padded to the largest count, one batched product
    x = s["x"] if s["rows"] is None else s["x"][s["rows"].long()]
    offsets, most = s["offsets"].long(), s["most"]
    r = x.shape[0]
    at = offsets[:-1, None] + torch.arange(most, device=x.device)
    held = at < offsets[1:, None]
    padded = torch.where(held.unsqueeze(-1), x[at.clamp_max(r - 1)].float(), 0.0)
    y = padded @ _dequantize(s["w"]).transpose(1, 2)
    return _activate(y[held], s["case"]["act"]).to(x.dtype)


def _plain_route(s):
    z, k = s["logits"].float(), s["case"]["top"]
    t, e = z.shape
    p = torch.exp(z - z.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    experts = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
    weights = p.gather(1, experts)
    if s["case"]["normalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    flat = experts.flatten()
    order = torch.sort(flat, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(t * k, device=z.device)
    offsets = torch.zeros(e + 1, dtype=torch.int64, device=z.device)
    offsets[1:] = torch.bincount(flat, minlength=e).cumsum(0)
    return [experts.int(), weights, (order // k).int(), slots.view(t, k).int(), offsets.int()]


def _plain_combine(s):
    y = (s["y"][s["slots"].long()].float() * s["weights"].unsqueeze(-1)).sum(1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["y"].dtype)


def run(state):
    case = state["case"]
    op, act = case["op"], case.get("act") or None
    if own:
        from chad_b200 import ops

        if op == "matmul":
            return ops.quantized_matmul(state["x"], state["w"], activation=act)
        if op == "grouped":
            return ops.grouped_quantized_matmul(state["x"], state["w"], state["offsets"], rows=state["rows"], activation=act)
        if op == "route":
            return list(ops.route_topk(state["logits"], case["top"], normalize=case["normalize"]))
        return ops.expert_combine(state["y"], state["slots"], state["weights"], residual=state["residual"])
    return {"matmul": _plain_matmul, "grouped": _plain_grouped, "route": _plain_route, "combine": _plain_combine}[op](state)


# ---------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------

def _values64(w):
    """Values of one weight matrix in 64 bits, from its bytes: low nibble first."""
    word, scale, bias = w
    by = word.contiguous().view(torch.uint8)
    codes = torch.stack((by % 16, torch.div(by, 16, rounding_mode="floor")), -1).flatten(-2).double()
    return torch.addcmul(bias.double().repeat_interleave(GROUP, -1), codes, scale.double().repeat_interleave(GROUP, -1))


def _product64(x, w, act):
    y = torch.einsum("mk,nk->mn", x.double(), _values64(w))
    if act:
        half = y.shape[1] // 2
        y = torch.nn.functional.silu(y[:, :half]) * y[:, half:]
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "matmul":
        return _product64(s["x"], s["w"], case["act"])
    if op == "grouped":
        x = s["x"] if s["rows"] is None else s["x"].index_select(0, s["rows"])
        ends = s["offsets"].tolist()
        parts = [_product64(x[a:b], [v[i] for v in s["w"]], case["act"]) for i, (a, b) in enumerate(zip(ends, ends[1:])) if b > a]
        return torch.cat(parts)
    if op == "route":
        p = torch.softmax(s["logits"].double(), -1)
        weights = p.sort(-1, descending=True).values[:, :case["top"]]
        if case["normalize"]:
            weights = weights / weights.sum(-1, keepdim=True)
        return [None, weights, None, None, None]
    y = torch.einsum("tkn,tk->tn", s["y"].double()[s["slots"].long()], s["weights"].double())
    return y if s["residual"] is None else y + s["residual"].double()
