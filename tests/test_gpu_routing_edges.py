"""Routing and the weighted sum at sizes and in processes where an earlier call could hide a fault."""

import os
import subprocess
import sys

import pytest
import torch

from chad_b200 import ops

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def fresh(code, *args):
    """Run a script in a process whose first library call is its own."""
    r = subprocess.run([sys.executable, "-c", code, *map(str, args)], cwd=ROOT, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("t,e,k", [(33000, 361, 2), (66000, 186, 3)])
def test_route_just_below_48_kib_of_masks_first(t, e, k):
    """Dynamic shared memory that passes the default bound only with the static bytes."""
    fresh("import sys, torch\n"
          "from tests.test_gpu_experts import check_route\n"
          "t, e, k = map(int, sys.argv[1:])\n"
          "gen = torch.Generator().manual_seed(t)\n"
          "check_route(torch.randn(t, e, generator=gen).to(torch.bfloat16).cuda(), k, True)\n", t, e, k)


def test_a_refused_launch_is_not_reported_by_the_next_call():
    """A call into an invalidated capture is refused with the CUDA error; the next one succeeds."""
    fresh("""
import torch
from chad_b200 import ops
from chad_b200._lib import QKVError
y = torch.ones(8, 64, dtype=torch.bfloat16, device="cuda")
slots = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
weights, out = torch.ones(4, 2, device="cuda"), torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
ops.expert_combine(y, slots, weights, out=out)
torch.cuda.synchronize()
stream, graph, said = torch.cuda.Stream(), torch.cuda.CUDAGraph(), ""
with torch.cuda.stream(stream):
    graph.capture_begin(capture_error_mode="thread_local")
    try:
        stream.synchronize()  # not allowed while capturing: the capture is invalid from here on
    except RuntimeError:
        pass
    try:
        ops.expert_combine(y, slots, weights, out=out)
    except QKVError as error:
        said = str(error)
    try:
        graph.capture_end()
    except RuntimeError:
        pass
assert "capture" in said and "unsupported shape" not in said, said
out.zero_()
ops.expert_combine(y, slots, weights, out=out)
torch.cuda.synchronize()
assert bool((out == 2).all())
""")


@pytest.mark.parametrize("t,k,n", [(1, 1, 1), (40, 3, 17), (3000, 2, 33), (700, 8, 264), (5000, 9, 1024)])
def test_weighted_sum_over_its_residual(t, k, n):
    """In place and apart are the same bits, at sizes where neighbouring threads share lines."""
    gen = torch.Generator().manual_seed(t + n)
    y = torch.randn(t * k, n, generator=gen).half().cuda()
    slots = torch.randperm(t * k, generator=gen).int().view(t, k).cuda()
    weights = torch.rand(t, k, generator=gen).cuda()
    residual = torch.randn(t, n, generator=gen).half().cuda()
    want = ops.expert_combine(y, slots, weights, residual=residual)
    for _ in range(4):
        over = residual.clone()
        assert ops.expert_combine(y, slots, weights, residual=over, out=over) is over
        assert torch.equal(over, want)


def test_first_calls_of_a_process_are_captured():
    """Shared-memory bounds, module loading and the status word need no call outside the capture."""
    fresh("""
import torch
from chad_b200 import ops
gen = torch.Generator().manual_seed(1)
def weights(*lead, k):
    return (torch.randint(-2 ** 31, 2 ** 31, (*lead, k // 8), generator=gen).int().cuda(),
            torch.rand(*lead, k // 64, generator=gen).bfloat16().cuda(),
            torch.randn(*lead, k // 64, generator=gen).bfloat16().cuda())
few, many = weights(4, 64, k=128), weights(4, 1000, k=512)
x, y = torch.randn(3, 128, generator=gen).bfloat16().cuda(), torch.randn(700, 512, generator=gen).bfloat16().cuda()
logits = torch.randn(700, 4, generator=gen).cuda()
def calls():
    r = ops.route_topk(logits, 2)
    return [ops.quantized_matmul(x, [t[0] for t in few]), ops.quantized_matmul(y, [t[0] for t in many]),
            *r, ops.grouped_quantized_matmul(y, many, r.offsets, rows=r.rows, activation="swiglu"),
            ops.expert_combine(torch.cat([y, y]), r.slots, r.weights, residual=y)]
graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
stream.wait_stream(torch.cuda.current_stream())
torch.cat([y, y])
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=stream):
    got = calls()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(got, calls()):
    assert torch.equal(a, b)
""")


def test_weighted_sum_of_slices_with_odd_rows():
    gen = torch.Generator().manual_seed(5)
    pool = torch.randn(30, 17, generator=gen).bfloat16().cuda()
    y, residual, out = pool[1:13], pool[13:17], torch.zeros(6, 17, dtype=torch.bfloat16, device="cuda")
    slots = torch.randperm(12, generator=gen).int().view(4, 3).cuda()
    weights = torch.rand(4, 3, generator=gen).cuda()
    ops.expert_combine(y, slots, weights, residual=residual, out=out[1:5])
    assert torch.equal(out[1:5], ops.expert_combine(y.clone(), slots, weights, residual=residual.clone()))
    assert bool((out[[0, 5]] == 0).all())
