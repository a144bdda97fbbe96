"""4-bit products where several calls, kernels or experts meet."""

import pytest
import torch

from chad_b200 import ops
from tests.test_gpu_matmul import check, make_weights, reference

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
