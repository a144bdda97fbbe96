"""Which products go to the kernel for many rows: it gathers rows into a workspace, the other none."""

import pytest

from chad_b200 import _lib


def takes_many(r, e, n, k):
    return _lib.load().qkv_matmul_workspace_size(r, e, n, k, 1) > 0


@pytest.mark.parametrize("r,n,k,many", [
    # as many rows as one pass over the weights has: 8, then 5, 2 and 1 of long K
    (8, 12288, 2048, False), (8, 12288, 8192, False), (9, 12288, 8192, True),
    (5, 12288, 14336, False), (6, 12288, 14336, True), (12, 8192, 14336, True), (12, 2048, 14336, False),
    (2, 8192, 28672, False), (4, 8192, 28672, False), (8, 8192, 28672, True), (8, 2048, 28672, False),
    (1, 8192, 65536, False), (4, 8192, 65536, True),
    # a row of x that does not fit beside the weights' stages
    (1, 64, 67392, False), (1, 64, 67456, True),
])
def test_one_matrix(r, n, k, many):
    assert takes_many(r, 1, n, k) == many


@pytest.mark.parametrize("e,n,k", [(128, 1536, 2048), (128, 2048, 768), (64, 1536, 2048), (8, 28672, 4096)])
def test_experts_by_their_average_rows(e, n, k):
    assert not takes_many(e * 8, e, n, k)
    assert not takes_many(e * 10, e, n, k)
    assert takes_many(e * 10 + 1, e, n, k)
    assert takes_many(e * 12, e, n, k)


def test_experts_of_long_k():
    # two rows a pass: as many passes as experts, a quarter more, and eight each
    assert not takes_many(16, 8, 8192, 28672)
    assert not takes_many(20, 8, 8192, 28672)
    assert takes_many(64, 8, 8192, 28672)
