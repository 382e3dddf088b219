"""A plan's usable_SM_count holds for the CTAs that share a windowed item, too."""
import pytest
import torch

from test_window_gpu import BF, E4, Case, _device_plan

pytestmark = pytest.mark.gpu


def _grids(call):
    """CTAs of the kernels that a call launches."""
    driver = pytest.importorskip("cuda.bindings.driver")
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    err, _, n = driver.cuGraphGetNodes(raw)
    assert err == driver.CUresult.CUDA_SUCCESS
    _, nodes, _ = driver.cuGraphGetNodes(raw, n)
    grids = []
    for node in nodes:
        _, kind = driver.cuGraphNodeGetType(node)
        if kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            err, p = driver.cuGraphKernelNodeGetParams(node)
            assert err == driver.CUresult.CUDA_SUCCESS
            grids.append(p.gridDimX * p.gridDimY * p.gridDimZ)
    return grids


@pytest.mark.parametrize("types", [(BF, BF), (BF, E4), (E4, E4)])
@pytest.mark.parametrize("tokens,hq", [(1, 8), (1, 16), (1, 64), (4, 32), (4, 64)])
@pytest.mark.parametrize("sms", [1, 3, 32, -1])
@pytest.mark.parametrize("device_made", [False, True])
def test_ctas_of_few_items(types, tokens, hq, sms, device_made):
    """Two CTAs an SM, and no fewer than there are items."""
    import msa_for_sail as msa
    c = Case([tokens] * 2, [4000, 3000], hq, 2, 2000, 4, "hnd", 128, *types)
    plan = _device_plan(c, tokens, 2 * tokens, usable_SM_count=sms) if device_made else c.plan(usable_SM_count=sms)
    out = torch.empty_like(c.q, dtype=torch.bfloat16)
    grids = _grids(lambda: msa.fmha_sail(c.q, c.k, c.v, plan, kv_indices=c.table, out=out))
    items = int(plan[3]["num_work"])
    assert grids and max(grids[:1]) <= max(2 * (148 if sms < 0 else sms), items)
    if sms < 0 and plan[3]["num_kv_splits"] == 1:
        assert grids[0] > items                                 # they do share items
    c.check(plan=plan)
