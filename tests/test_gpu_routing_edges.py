"""Routing and the weighted sum at sizes and in processes where an earlier call could hide a fault."""

import os
import subprocess
import sys

import pytest

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
