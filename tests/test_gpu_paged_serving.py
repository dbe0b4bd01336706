"""The operators of paged serving together, as a server calls them: prompts in chunks, requests of different lengths that decode, drafts that
are verified, pages that go back."""
import pytest
import torch

from gpu_ipc_example_b200 import Communicator
from gpu_ipc_example_b200.models.llama import LlamaConfig, LlamaTP, dense_decode_reference
from gpu_ipc_example_b200.models.paged import PagedCache, PagedCacheError

pytestmark = pytest.mark.gpu


def ints(v, dt=torch.int32):
    return torch.tensor(v, dtype=dt, device="cuda")


def served(model, prompts, chunks, cache):
    """Hidden states of every prompt's tokens, fed in the given pieces: chunks[i] is a list of lengths for prompt i, one for each step."""
    at, got = [0] * len(prompts), [[] for _ in prompts]
    for step in range(max(map(len, chunks))):
        new = [c[step] if step < len(c) else 0 for c in chunks]
        tokens = torch.cat([p[a:a + n] for p, a, n in zip(prompts, at, new)] + [prompts[0].new_zeros(3)])  # three rows without a token
        batch = cache.extend(ints(new), tokens.numel(), max(new))
        hidden = model.forward_paged(tokens, batch, cache)
        cache.check()
        for i, n in enumerate(new):
            got[i].append(hidden[0][sum(new[:i]):sum(new[:i + 1])].float().clone())
            at[i] += n
    return [torch.cat(g) for g in got]


@pytest.mark.parametrize("world,fusion", [(1, "gemm"), (2, "allreduce"), (2, "gemm")])
@pytest.mark.parametrize("page", [16, 64])
def test_prompts_in_chunks_match_the_dense_decoder(world, fusion, page):
    cfg = LlamaConfig.tiny128()
    with Communicator.virtual(world, 0, staging_bytes=64 << 20) as comm:
        model = LlamaTP(cfg, comm, batch=1, max_ctx=8, fusion=fusion, seed=3)
        g = torch.Generator(device="cuda").manual_seed(6)
        lens = [37, 5, 20]
        prompts = [torch.randint(0, cfg.vocab, (n,), device="cuda", generator=g) for n in lens]
        cache = PagedCache(model, requests=3, max_len=64, pages=12, page=page)
        # a whole prompt, single tokens, pieces of uneven lengths with pauses
        got = served(model, prompts, [[37], [1, 1, 1, 1, 1], [3, 0, 9, 1, 7]], cache)
        comm.check()
        assert cache.lens.tolist() == lens
        for p, x in zip(prompts, got):
            want = torch.stack([y[0] for y in dense_decode_reference(model, [t.view(1) for t in p])])
            torch.testing.assert_close(x, want, atol=6e-2, rtol=5e-2)  # as the decoder's own tests
        cache.trim(torch.zeros_like(cache.lens))
        cache.check()
        assert int(cache.n_free) == 12 and sorted(cache.free_pages.tolist()) == list(range(12))


def test_speculative_steps_leave_what_was_accepted():
    """Drafts are verified, the turned down ones leave the cache, and what follows is computed as if they never had been there."""
    cfg = LlamaConfig.tiny128()
    with Communicator.virtual(2, 0, staging_bytes=64 << 20) as comm:
        model = LlamaTP(cfg, comm, batch=1, max_ctx=8, fusion="allreduce", seed=4)
        g = torch.Generator(device="cuda").manual_seed(8)
        B, K = 3, 4
        prompts = [torch.randint(0, cfg.vocab, (n,), device="cuda", generator=g) for n in (17, 3, 9)]
        cache = PagedCache(model, requests=B, max_len=128, pages=24, page=16)
        served(model, [p[:-1] for p in prompts], [[16], [2], [8]], cache)
        text = [p.tolist() for p in prompts]
        for step in range(4):
            last = ints([t[-1] for t in text], torch.int64)
            draft_probs = torch.softmax(torch.randn(B, K, cfg.vocab, device="cuda", generator=g), -1)
            drafts = torch.multinomial(draft_probs.view(B * K, -1), 1, generator=g).view(B, K)
            accept = torch.rand(B, K, device="cuda", generator=g) * (0.2 if step % 2 else 1.0)  # many accepted, and few
            tokens, accepted = model.verify(last, drafts, draft_probs, cache, accept, torch.rand(B, device="cuda", generator=g))
            cache.check()
            comm.check()
            for i in range(B):
                n = int(accepted[i])
                assert tokens[i, :n].tolist() == drafts[i, :n].tolist() and tokens[i, n + 1:].tolist() == [-1] * (K - n)
                assert 0 <= int(tokens[i, n]) < cfg.vocab
                text[i] += tokens[i, :n + 1].tolist()
            assert cache.lens.tolist() == [len(t) - 1 for t in text]
            held = sum((len(t) - 1 + 15) // 16 for t in text)
            assert int(cache.n_free) == 24 - held
        batch = cache.extend(ints([1] * B), B, 1)
        hidden = model.forward_paged(ints([t[-1] for t in text], torch.int64), batch, cache)[0].float()
        cache.check()
        for i, t in enumerate(text):
            want = dense_decode_reference(model, [ints([x], torch.int64) for x in t])[-1][0]
            torch.testing.assert_close(hidden[i], want, atol=6e-2, rtol=5e-2)


def test_a_step_without_room_changes_nothing():
    cfg = LlamaConfig.tiny128()
    with Communicator.virtual(1, 0, staging_bytes=64 << 20) as comm:
        model = LlamaTP(cfg, comm, batch=1, max_ctx=8, fusion="allreduce")
        cache = PagedCache(model, requests=2, max_len=64, pages=3, page=16)
        tokens = torch.arange(40, device="cuda")
        batch = cache.extend(ints([30, 10]), 40)
        model.forward_paged(tokens, batch, cache)
        cache.check()
        state = lambda: (cache.k[0][0].view(torch.int16), cache.v[0][1].view(torch.int16), cache.block_table, cache.lens, cache.free_pages, cache.n_free)  # bits: unused places hold anything
        keep = [c.clone() for c in state()]
        batch = cache.extend(ints([10, 1]), 11)  # a page more than there is
        model.forward_paged(tokens[:11], batch, cache)
        drafts = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
        model.verify(tokens[:2], drafts, None, cache, torch.rand(2, 3, device="cuda"), torch.rand(2, device="cuda"))
        with pytest.raises(PagedCacheError, match="pages run out"):
            cache.check()
        assert all(torch.equal(a, b) for a, b in zip(keep, state()))
        cache.check()  # said once


def test_a_captured_step_serves_every_length():
    cfg = LlamaConfig.tiny128()
    with Communicator.virtual(1, 0, staging_bytes=64 << 20) as comm:
        model = LlamaTP(cfg, comm, batch=1, max_ctx=8, fusion="allreduce", seed=5)
        g = torch.Generator(device="cuda").manual_seed(1)
        prompts = [torch.randint(0, cfg.vocab, (n,), device="cuda", generator=g) for n in (25, 1, 40)]
        eager = PagedCache(model, requests=3, max_len=128, pages=20, page=16)
        cache = PagedCache(model, requests=3, max_len=128, pages=20, page=16)
        served(model, prompts, [[25], [1], [40]], eager)
        served(model, prompts, [[25], [1], [40]], cache)
        new, tokens = ints([1, 1, 1]), torch.zeros(3, dtype=torch.int64, device="cuda")
        steps = [torch.randint(0, cfg.vocab, (3,), device="cuda", generator=g) for _ in range(20)]
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            tokens.copy_(steps[0])
            model.forward_paged(tokens, cache.extend(new, 3, 1), cache)  # warms up; the step that it made goes away again
            cache.trim(ints([25, 1, 40]))
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = model.forward_paged(tokens, cache.extend(new, 3, 1), cache)[0]
            for t in steps:
                tokens.copy_(t)
                graph.replay()
                want = model.forward_paged(t, eager.extend(new, 3, 1), eager)[0]
                stream.synchronize()
                assert torch.equal(out, want)
        cache.check()
        eager.check()
        assert cache.lens.tolist() == eager.lens.tolist() == [45, 21, 60]


@pytest.mark.parametrize("max_new", [1, 20])  # of the kernel for few rows, and of the other
def test_more_new_tokens_than_announced_are_said(max_new):
    cfg = LlamaConfig.tiny128()
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        model = LlamaTP(cfg, comm, batch=1, max_ctx=8, fusion="gemm", seed=5)
        cache = PagedCache(model, requests=2, max_len=128, pages=12, page=32)
        tokens = torch.arange(42, device="cuda")
        model.forward_paged(tokens, cache.extend(ints([2, 40]), 42, max_new), cache)
        with pytest.raises(PagedCacheError, match="more new tokens than max_new"):
            cache.check()
        cache.trim(ints([0, 0]))
        got = model.forward_paged(tokens, cache.extend(ints([2, 40]), 42, 40), cache)[0].clone()
        cache.check()
        cache.trim(ints([0, 0]))
        assert torch.equal(got, model.forward_paged(tokens, cache.extend(ints([2, 40]), 42), cache)[0])
        cache.check()


def test_a_captured_step_outlives_larger_steps():
    """The scratch that a captured step of single tokens uses is the one that a long prompt takes later."""
    cfg = LlamaConfig.tiny128()
    with Communicator.virtual(1, 0, staging_bytes=16 << 20) as comm:
        model = LlamaTP(cfg, comm, batch=1, max_ctx=8, fusion="allreduce", seed=5)
        cache = PagedCache(model, requests=2, max_len=512, pages=24, page=64)
        tokens, one = torch.tensor([3, 4], device="cuda"), ints([1, 1])

        def step():
            return model.forward_paged(tokens, cache.extend(one, 2, 1), cache)[0]

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = step()
            where = cache.workspace.data_ptr()
            for rep in range(2):
                cache.trim(ints([0, 0]))
                model.forward_paged(torch.arange(400, device="cuda") % cfg.vocab, cache.extend(ints([100, 300]), 400, 300), cache)
                graph.replay()
                got = out.clone()
                cache.trim(ints([100, 300]))
                assert torch.equal(got, step())
            cache.check()
            comm.check()
            assert cache.workspace.data_ptr() == where
        torch.cuda.synchronize()


def test_refusals():
    cfg = LlamaConfig.tiny()
    with Communicator.virtual(1, 0, staging_bytes=64 << 20) as comm:
        with pytest.raises(ValueError, match="decode kernels"):
            PagedCache(LlamaTP(cfg, comm, batch=1, max_ctx=8), requests=1, max_len=8, pages=1)
        with pytest.raises(ValueError, match="16, 32, 64 or 128"):
            PagedCache(LlamaTP(LlamaConfig.tiny128(), comm, batch=1, max_ctx=8), requests=1, max_len=8, pages=1, page=24)
