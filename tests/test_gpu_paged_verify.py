"""Speculative steps of the decoder where not every request takes part, has all drafts or finds room, and where the call is refused."""
import io
import threading

import pytest
import torch

import paged_reference as ref
from gpu_ipc_example_b200 import Communicator
from gpu_ipc_example_b200._ext import load
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
                       dict(temperature=0.0), dict(temperature=float("nan")), dict(draft_lens=ints([1, 1, 1])), dict(draft_lens=ints([1, 1], torch.int64))):
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


@pytest.mark.parametrize("certain", [False, True])
def test_requests_with_fewer_drafts_and_without_any_part(certain):
    """Slot 1 has no request, slot 2 has room for two tokens and one draft, slot 4 none at all, slot 5 sits the step out."""
    lens, count = [17, 0, 62, 9, 16, 33], [K, -1, 1, 2, 0, -1]
    with Communicator.virtual(2, 0, staging_bytes=64 << 20) as comm:
        prompts = [n if n else 1 for n in lens]
        (model, cache, g), (_, other, _) = made(comm, prompts), made(comm, prompts)
        for c in (cache, other):
            c.trim(ints(lens))  # slot 1: a request that is done
        last, drafts, probs, accept, sample = numbers(model, 6, g)
        padded, told = drafts.clone(), last.clone()
        for i, n in enumerate(count):
            padded[i, max(n, 0):] = -1  # whatever stands there
            if n < 0:
                told[i] = -1
        p = None if certain else probs
        counts = ints([x for n in count for x in (n, 7)])[::2]  # strided
        tokens, accepted = model.verify(told, padded, p, cache, accept, sample, draft_lens=counts)
        cache.check()
        comm.check()
        # the same by hand: the tokens of the requests that take part, one request after the other
        ids = [torch.cat([last[i:i + 1], drafts[i, :n]]) if n >= 0 else last[:0] for i, n in enumerate(count)]
        batch = other.extend(ints([len(x) for x in ids]), 6 * (K + 1), K + 1)
        hidden = model.forward_paged(torch.cat(ids + [last.new_zeros(6 * (K + 1) - sum(map(len, ids)))]), batch, other)
        flat = model.probabilities(hidden).cpu()
        at, target = 0, torch.zeros(6, K + 1, model.cfg.vocab)
        for i, x in enumerate(ids):
            target[i, :len(x)] = flat[at:at + len(x)]
            at += len(x)
        want, n_want = ref.verify(target, None if certain else probs.cpu(), drafts.cpu(), ints(count).cpu(), accept.cpu(), sample.cpu())
        for i, n in enumerate(count):
            if n < 0:
                want[i], n_want[i] = -1, -1
        assert torch.equal(tokens.cpu(), want) and torch.equal(accepted.cpu(), n_want)
        assert cache.lens.tolist() == [n + a + 1 for n, a in zip(lens, n_want.tolist())]
        assert int(cache.n_free) == 20 - sum(ref.pages_of(n, 16) for n in cache.lens.tolist())


@pytest.mark.parametrize("world,fusion", [(1, "gemm"), (2, "gemm"), (2, "allreduce")])
def test_steps_without_drafts_and_without_requests(world, fusion):
    """No drafts at all: a word is drawn for every request.  No request that takes part: nothing happens.  Numbers outside of -1 .. K are cut off."""
    with Communicator.virtual(world, 0, staging_bytes=64 << 20) as comm:
        model = LlamaTP(LlamaConfig.tiny128(), comm, batch=1, max_ctx=8, fusion=fusion, seed=4)
        cache = PagedCache(model, requests=3, max_len=64, pages=20, page=16)
        g = torch.Generator(device="cuda").manual_seed(8)
        served(model, [torch.randint(0, model.cfg.vocab, (n,), device="cuda", generator=g) for n in (5, 1, 20)], [[5], [1], [20]], cache)
        last, drafts, probs, accept, sample = numbers(model, 3, g)
        before = tables(cache)
        tokens, accepted = model.verify(last, drafts, probs, cache, accept, sample, draft_lens=ints([-1, -1, -1]))
        assert (tokens == -1).all() and (accepted == -1).all() and all(torch.equal(a, b) for a, b in zip(before, tables(cache)))
        tokens, accepted = model.verify(last, drafts[:, :0], None, cache, accept[:, :0], sample)
        assert accepted.tolist() == [0] * 3 and all(0 <= t < model.cfg.vocab for t in tokens[:, 0].tolist()) and cache.lens.tolist() == [6, 2, 21]
        tokens, accepted = model.verify(last, drafts, None, cache, torch.zeros_like(accept), sample, draft_lens=ints([-7, 99, 1]))
        assert accepted.tolist() == [-1, K, 1] and cache.lens.tolist() == [6, 2 + K + 1, 23]
        assert tokens[1, :K].tolist() == drafts[1].tolist() and tokens[0].tolist() == [-1] * (K + 1)
        cache.check()
        comm.check()


def test_a_captured_speculative_step():
    """Draft lengths change between the replays, and the pages run out in the end."""
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        (model, cache, g), (_, other, _) = made(comm, [5, 30, 12], pages=7), made(comm, [5, 30, 12], pages=7)
        args, count = numbers(model, 3, g), ints([K, 0, -1])
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        refused = 0
        with torch.cuda.stream(stream):
            before = cache.lens.clone()
            model.verify(*args[:3], cache, *args[3:], draft_lens=count)
            cache.trim(before)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                got = model.verify(*args[:3], cache, *args[3:], draft_lens=count)
            for step in range(40):
                for a, b in zip(args, numbers(model, 3, g)):
                    a.copy_(b)
                count.copy_(ints([step % (K + 2) - 1, K, (step + 2) % (K + 2) - 1]))
                graph.replay()
                want = model.verify(*args[:3], other, *args[3:], draft_lens=count)
                stream.synchronize()
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
                assert torch.equal(cache.lens, other.lens)
                refused += bool((want[1] == -1).all())
        assert refused
        with pytest.raises(PagedCacheError, match="pages run out"):
            cache.check()
        del graph


def test_a_small_cache_takes_padded_batches():
    """Fewer tokens fit the cache than the batch has rows: the rows say nothing of how long a request is."""
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        model = LlamaTP(LlamaConfig.tiny128(), comm, batch=1, max_ctx=8, fusion="allreduce", seed=3)
        tokens = torch.arange(40, device="cuda")
        hidden = []
        for max_len in (8, 4000):
            cache = PagedCache(model, requests=1, max_len=max_len, pages=4, page=16)
            hidden.append(model.forward_paged(tokens, cache.extend(ints([8]), 40), cache)[0][:8].clone())
            cache.check()
        torch.testing.assert_close(hidden[0].float(), hidden[1].float(), atol=6e-2, rtol=5e-2)  # another kernel, perhaps


def test_what_extend_returns_has_memory_of_its_own():
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        model, cache, _ = made(comm, [7, 20])
        batch = cache.extend(ints([3, 1]), 6, 3)
        out = (batch.cu_new, batch.slots, batch.positions)
        want = [t.tolist() for t in out]
        assert len({t.untyped_storage().data_ptr() for t in out}) == 3
        file = io.BytesIO()
        torch.save(out, file)
        file.seek(0)
        assert [t.tolist() for t in torch.load(file)] == want
        status = torch.ops.b200ipc.paged_extend(cache.block_table, cache.lens, ints([0, 0]), cache.free_pages, cache.n_free, 16, 1)[3]
        status.resize_(64).fill_(-5)
        assert [t.tolist() for t in out] == want


@pytest.mark.parametrize("few,many", [(4200, 8192), (6500, 8192)])  # above 48 KB of shared memory for extend alone, and for trim as well
def test_threads_with_different_numbers_of_requests(few, many):
    """Launches of both sizes from two host threads: what one of them asks of the kernel does not take from the other."""
    failed = []

    def steps(requests):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                table, lens, none = torch.full((requests, 1), -1, dtype=torch.int32, device="cuda"), ints([0] * requests), ints([0] * requests)
                free, n_free = torch.arange(requests, dtype=torch.int32, device="cuda"), ints([requests])
                for i in range(20000):
                    if i % 2:
                        torch.ops.b200ipc.paged_trim(table, lens, none, free, n_free, 16)
                    else:
                        torch.ops.b200ipc.paged_extend(table, lens, none, free, n_free, 16, 1)
                    if i % 500 == 0:
                        torch.cuda.current_stream().synchronize()
        except Exception as e:  # of a thread
            failed.append(e)

    load()
    threads = [threading.Thread(target=steps, args=(n,)) for n in (few, many)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]
