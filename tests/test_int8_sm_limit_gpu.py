"""The 8-bit product keeps to the limit on the GEMMs' SMs, whichever kernel takes it, with the same results."""

from __future__ import annotations

import pytest
import torch

from ats_v2_b200 import _lib
from ats_v2_b200.quantization import int8_linear, quantize_int8

pytestmark = pytest.mark.gpu


def grids(graph):
    """Blocks of each kernel of a captured graph, in no particular order."""
    from cuda.bindings import driver

    def ok(result):
        assert result[0] == driver.CUresult.CUDA_SUCCESS, result[0]
        return result[1:]

    handle = driver.CUgraph(graph.raw_cuda_graph())
    count = ok(driver.cuGraphGetNodes(handle))[-1]
    nodes = ok(driver.cuGraphGetNodes(handle, count))[0]
    params = [ok(driver.cuGraphKernelNodeGetParams(n))[0] for n in nodes]
    return [p.gridDimX * p.gridDimY * p.gridDimZ for p in params]


@pytest.mark.parametrize("limit", [1, 2, 37, 100, 147])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (1, 600, 17000), (8, 4096, 4096), (48, 11008, 4096), (40, 256, 2048),
                                   (200, 2048, 8192), (2304, 4096, 512)])
def test_the_product_keeps_to_the_limit(M, N, K, limit):
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).cuda().bfloat16()
    w, s = quantize_int8(torch.randn(N, K, generator=g).cuda())
    want = int8_linear(x, w, s)
    with _lib.gemm_sm_limit(limit):
        assert torch.equal(int8_linear(x, w, s), want)
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            int8_linear(x, w, s)
    blocks = grids(graph)
    # the quantisation of rows of up to 2048 takes four rows to a block, of longer ones one; one token of up to 16384 none
    alone = M == 1 and K <= 16384
    if not alone:
        blocks.remove(-(-M // 4) if K <= 2048 else M)
    assert len(blocks) == 1 and blocks[0] <= max(limit, 1 if alone else 2)  # a pair of CTAs is the least of the others
