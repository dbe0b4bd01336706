"""What of paged serving needs no GPU: a time limit that is refused, probabilities of several processes."""
import multiprocessing as mp

import pytest
import torch

from gpu_ipc_example_b200.models.llama import LlamaTP
from test_paged_cpu import attention_args, ops


@pytest.mark.parametrize("timeout_ms", [0, -1, 60001])
def test_attention_refuses_a_time_limit(timeout_ms):
    with pytest.raises(RuntimeError, match="timeout_ms"):
        ops().paged_attention(**attention_args(), timeout_ms=timeout_ms)


def head(rank, world):
    """The decoder's head alone: rank's share of the vocabulary."""
    g = torch.Generator().manual_seed(rank)
    model = LlamaTP.__new__(LlamaTP)
    model.world, model.nlocal = world, 1
    model.lm_head = [torch.randn(96, 64, generator=g).bfloat16()]
    return model


def hidden():
    return torch.randn(5, 64, generator=torch.Generator().manual_seed(77)).bfloat16()


def probabilities_of_a_rank(rank, world, file, queue):
    import torch.distributed as dist

    dist.init_process_group("gloo", init_method=f"file://{file}", rank=rank, world_size=world)
    p = head(rank, world).probabilities([hidden()], 0.7)
    queue.put((rank, p.tolist()))
    dist.barrier()
    dist.destroy_process_group()


def test_probabilities_of_two_processes(tmp_path):
    """Each has half of the vocabulary and gets the whole of it."""
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    ranks = [ctx.Process(target=probabilities_of_a_rank, args=(r, 2, str(tmp_path / "store"), queue)) for r in range(2)]
    for p in ranks:
        p.start()
    got = dict(queue.get(timeout=240) for _ in ranks)
    for p in ranks:
        p.join(60)
        assert p.exitcode == 0
    logits = torch.cat([hidden() @ head(r, 2).lm_head[0].t() for r in range(2)], -1)
    want = torch.softmax(logits.double() / 0.7, -1)
    for r in range(2):
        # exponent and sum in fp32: a few units of 2^-24 for each of logit / 0.7 (below 64 in size: 2^-18), exponential and quotient
        torch.testing.assert_close(torch.tensor(got[r], dtype=torch.float64), want, rtol=2.0 ** -16, atol=0)


@pytest.mark.parametrize("temperature", [0, 0.0, -1.0, float("nan")])
def test_probabilities_refuse_a_temperature(temperature):
    with pytest.raises(ValueError, match="temperature"):
        head(0, 1).probabilities([hidden()], temperature)
