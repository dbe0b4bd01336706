"""Speculative steps of the decoder where not every request takes part, has all drafts or finds room, and where the call is refused."""

import pytest
import torch

from gpu_ipc_example_b200 import Communicator
from gpu_ipc_example_b200.models.llama import LlamaConfig, LlamaTP
from gpu_ipc_example_b200.models.paged import PagedCache, PagedCacheError
from test_gpu_paged_serving import ints, served

pytestmark = pytest.mark.gpu
K = 3


def state(cache):
    """Bits of all that a step changes; what stands behind a request's last token is of no account, but unchanged where nothing is written."""
    return [c.clone() for c in (cache.k[0][0].view(torch.int16), cache.v[0][1].view(torch.int16), cache.block_table, cache.lens, cache.free_pages, cache.n_free)]


def tables(cache):
    return [c.clone() for c in (cache.block_table, cache.lens, cache.free_pages, cache.n_free)]


def made(comm, prompts, max_len=64, pages=20, seed=4):
    model = LlamaTP(LlamaConfig.tiny128(), comm, batch=1, max_ctx=8, fusion="allreduce", seed=seed)
    cache = PagedCache(model, requests=len(prompts), max_len=max_len, pages=pages, page=16)
    g = torch.Generator(device="cuda").manual_seed(8)
    text = [torch.randint(0, model.cfg.vocab, (n,), device="cuda", generator=g) for n in prompts]
    served(model, text, [[n] for n in prompts], cache)
    return model, cache, g


def numbers(model, B, g):
    """last, drafts, their probabilities, accept, sample"""
    probs = torch.softmax(torch.randn(B, K, model.cfg.vocab, device="cuda", generator=g), -1)
    drafts = torch.multinomial(probs.view(B * K, -1), 1, generator=g).view(B, K)
    last = torch.randint(0, model.cfg.vocab, (B,), device="cuda", generator=g)
    return [last, drafts, probs, torch.rand(B, K, device="cuda", generator=g) * 0.5, torch.rand(B, device="cuda", generator=g)]


def test_a_step_without_room_answers_nothing():
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        model, cache, g = made(comm, [30, 10], pages=3)
        keep = state(cache)
        last, drafts, probs, accept, sample = numbers(model, 2, g)
        for p in (probs, None):
            tokens, accepted = model.verify(last, drafts, p, cache, torch.zeros_like(accept), sample)  # all drafts would be accepted
            assert (tokens == -1).all() and (accepted == -1).all()
            assert all(torch.equal(a, b) for a, b in zip(keep, state(cache)))
        with pytest.raises(PagedCacheError, match="pages run out"):
            cache.check()


def test_refused_arguments_leave_the_cache_as_it_is():
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        model, cache, g = made(comm, [7, 20])
        keep = tables(cache)
        last, drafts, probs, accept, sample = numbers(model, 2, g)
        good = dict(last=last, drafts=drafts, draft_probs=probs, cache=cache, accept=accept, sample=sample)
        for change in (dict(draft_probs=probs.half()), dict(draft_probs=probs[:, :2]), dict(draft_probs=probs[..., :100]), dict(draft_probs=probs.transpose(1, 2)),
                       dict(accept=accept.double()), dict(accept=accept[:, :2]), dict(sample=sample[:1]), dict(sample=sample.cpu()), dict(last=last[:1]),
                       dict(last=last.float()), dict(drafts=drafts.int()), dict(drafts=drafts[0]), dict(drafts=drafts[:1], draft_probs=None, accept=accept[:1]),
                       dict(temperature=0.0), dict(temperature=float("nan"))):
            with pytest.raises((ValueError, RuntimeError)):
                model.verify(**{**good, **change})
            assert all(torch.equal(a, b) for a, b in zip(keep, tables(cache))), change.keys()
        with pytest.raises(ValueError, match="temperature"):
            model.probabilities([torch.zeros(1, model.cfg.hidden, device="cuda", dtype=model.cfg.dtype)], 0.0)
        cache.check()


def test_a_step_that_fails_midway_leaves_no_tokens(monkeypatch):
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        model, cache, g = made(comm, [7, 20])
        keep = tables(cache)
        args = numbers(model, 2, g)

        def fails(*_):
            raise torch.OutOfMemoryError("no memory for the probabilities")

        monkeypatch.setattr(model, "probabilities", fails)
        with pytest.raises(torch.OutOfMemoryError):
            model.verify(*args[:3], cache, *args[3:])
        assert all(torch.equal(a, b) for a, b in zip(keep, tables(cache)))
        cache.check()
