"""Waits inside the paged attention that run out: a CTA's first copies are left out.  The kernels return, the workspace says so, and the next
call is right: shared and tensor memory were given back."""
import pytest
import torch

from gpu_ipc_example_b200 import Communicator
from gpu_ipc_example_b200.models.llama import LlamaConfig, LlamaTP
from gpu_ipc_example_b200.models.paged import PagedCache, PagedCacheError
from test_gpu_paged import D, ints, ops, paged_problem, workspace

pytestmark = pytest.mark.gpu
MUTE_SENDS = 2


# One request in one span (1), one in many pieces, several items a span; requests of up to 16 rows, of up to 128, of more
@pytest.mark.parametrize("have,new", [([300], [1]), ([6000], [2]), ([900] * 160, [1] * 160), ([300], [5]), ([6000], [5]), ([2000], [300]), ([700] * 40, [40] * 40)])
def test_copies_that_never_come(have, new):
    """The first copies of one CTA are left out: the waits for them end, the kernel leaves and says so, and the next call is right."""
    hq = 8
    p = paged_problem(torch.bfloat16, 32, hq, 1, have, new)
    q, k, v, table, total, cu = p
    ws = workspace(hq, 1, max(new))
    args = (q, k, v, ints(table), ints(total), ints(cu), ws, hq, 1, max(new))
    want = ops().paged_attention(*args)
    out = ops().paged_attention(*args, timeout_ms=20, flags=MUTE_SENDS)
    torch.cuda.synchronize()
    assert out.shape == want.shape and int(ws[:4].view(torch.int32)) == 1
    ws.zero_()
    for _ in range(3):
        assert torch.equal(ops().paged_attention(*args), want)
    assert int(ws[:4].view(torch.int32)) == 0


@pytest.mark.parametrize("new", [[1, 1], [30, 1]])
def test_a_paged_cache_says_that_a_wait_ran_out(new):
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        model = LlamaTP(LlamaConfig.tiny128(), comm, batch=1, max_ctx=8, fusion="allreduce", seed=5)
        cache = PagedCache(model, requests=2, max_len=64, pages=8, page=16)
        tokens = torch.arange(sum(new), device="cuda")

        def step():
            cache.trim(torch.zeros_like(cache.lens))
            batch = cache.extend(ints(new), sum(new), max(new))
            return model.forward_paged(tokens, batch, cache)[0].clone(), batch

        want, batch = step()
        cache.check()
        q = torch.zeros(sum(new), model.hq * D, device="cuda", dtype=model.cfg.dtype)
        ops().paged_attention(q, cache.k[0][0], cache.v[0][0], cache.block_table, cache.lens, batch.cu_new, cache.workspace, model.hq, model.hkv,
                                   batch.max_new, 20, MUTE_SENDS)
        with pytest.raises(PagedCacheError, match="wait inside the attention ran out"):
            cache.check()
        for _ in range(2):
            assert torch.equal(step()[0], want)
        cache.check()
