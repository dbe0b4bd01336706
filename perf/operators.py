"""What is timed of the operators of paged serving: a cache of keys and values cut into pages, what fills and reads it, and the
verification of drafted tokens.

A step of a server that has requests of different lengths in one batch takes them in this order, and the kinds below are its parts:

  tables     the block table grows by the pages that the new tokens need (`paged_extend`, with slots and positions of the tokens),
             and shrinks again by what is given up (`paged_trim`): 1 - 1024 requests, 1 - 32768 new tokens, pages of 16 - 128
  append     rotary positions of the new tokens' queries and keys, keys and values into their pages (`rope_paged_append`):
             1 - 8192 tokens, 1 - 8 KV heads, 1 - 8 query heads for each
  attention  the new tokens over the cache, themselves included (`paged_attention`): 1 - 96 requests with 1 - 4096 new tokens each and
             up to 32768 in the cache
  verify     drafted tokens against the target's probabilities, and the token behind the accepted ones (`verify_drafts`):
             1 - 64 requests, 1 - 8 drafts, 2048 - 128256 words

Heads have 128 dimensions, as in the decoder; head counts are its per-rank shapes (8 query heads on one KV head) and the unsharded ones.
Activations are N(0, 1), as those that the other cases and the tests have.  Lengths belong to the case and values to the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_D = 128
_THETA = 5e5


def listed():
    return [
        # every step of a decoding server: one token for each of 32 requests, most of them without a new page
        dict(name="tables 32 x 1", kind="tables", requests=32, lo=1, hi=1, context=2048, page=64, shape=1),
        # a step that takes in prompts: 512 requests, some without new tokens, 1 - 64 tokens for the others
        dict(name="tables 512 ragged", kind="tables", requests=512, lo=0, hi=64, context=4096, page=16, shape=2),
        # decoding: 32 tokens of the per-rank shape
        dict(name="append 32", kind="append", tokens=32, hq=8, hkv=1, context=2048, page=64, pad=0, dtype="fp16", shape=3),
        # prompts, all heads on one GPU, in a batch that is padded, far into long contexts
        dict(name="append 4001", kind="append", tokens=4001, hq=64, hkv=8, context=100000, page=16, pad=95, dtype="bf16", shape=4),
        # one user, one token: the smallest call
        dict(name="attention 1 x 300", kind="attention", requests=1, lo=1, hi=1, clo=300, chi=300, chunk=0, hq=8, hkv=1, page=16,
             dtype="fp16", shape=5),
        # the decoder's step of 32 requests around 2048 tokens
        dict(name="attention 32 x 2048", kind="attention", requests=32, lo=1, hi=1, clo=1900, chi=2200, chunk=0, hq=8, hkv=1, page=64,
             dtype="fp16", shape=6),
        # long documents of very different lengths, one token each
        dict(name="attention 16 x 32768", kind="attention", requests=16, lo=1, hi=1, clo=1000, chi=32768, chunk=0, hq=16, hkv=2, page=64,
             dtype="bf16", shape=7),
        # four drafts behind the last token of every request
        dict(name="attention drafts 24 x 5", kind="attention", requests=24, lo=5, hi=5, clo=500, chi=8192, chunk=0, hq=16, hkv=2, page=32,
             dtype="bf16", shape=8),
        # a chunk of a long prompt, per-rank shape
        dict(name="attention chunk 512", kind="attention", requests=1, lo=512, hi=512, clo=16384, chi=16384, chunk=0, hq=8, hkv=1, page=64,
             dtype="fp16", shape=9),
        # a chunk of one prompt among requests that decode
        dict(name="attention mixed", kind="attention", requests=24, lo=0, hi=1, clo=200, chi=6000, chunk=2047, hq=32, hkv=8, page=128,
             dtype="bf16", shape=10),
        # whole prompts of different lengths
        dict(name="attention prompts", kind="attention", requests=4, lo=1500, hi=4096, clo=0, chi=0, chunk=0, hq=32, hkv=8, page=64,
             dtype="fp16", shape=11),
        # four drafts of 32 requests over the decoder's vocabulary
        dict(name="verify 32 x 4", kind="verify", requests=32, drafts=4, vocab=128256, shape=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attention", "attention", "attention", "verify"])
    page, dtype, shape = rng.choice([16, 32, 64, 128]), rng.choice(["fp16", "bf16"]), rng.randrange(1 << 20)
    if kind == "tables":
        n = _log(rng, 1, 1024)
        return dict(kind=kind, requests=n, lo=rng.choice([0, 1]), hi=_log(rng, 1, max(1, 32768 // n)), context=_log(rng, 16, 8192), page=page, shape=shape)
    hkv = rng.choice([1, 2, 4, 8])
    if kind == "append":
        return dict(kind=kind, tokens=_log(rng, 1, 8192 // hkv), hq=hkv * rng.choice([1, 2, 4, 5, 8]), hkv=hkv, context=_log(rng, 16, 100000),
                    page=page, pad=rng.choice([0, 0, 7, 64]), dtype=dtype, shape=shape)
    if kind == "verify":
        return dict(kind=kind, requests=_log(rng, 1, 64), drafts=rng.randint(1, 8), vocab=_log(rng, 2048, 128256), shape=shape)
    c = dict(kind=kind, hkv=hkv, hq=hkv * rng.choice([1, 2, 4, 5, 8]), page=page, dtype=dtype, shape=shape, chunk=0)
    what = rng.choice(["decode", "drafts", "chunk", "mixed", "prompts"])
    if what in ("decode", "drafts"):
        n = _log(rng, 1, 64)
        most = max(64, min(32768, (1 << 20) // (n * hkv)))
        new = 1 if what == "decode" else rng.randint(2, 8)
        c.update(requests=n, lo=new, hi=new, clo=_log(rng, 1, most), chi=most)
    elif what == "chunk":
        new = _log(rng, 65, 2048)
        most = max(64, min(32768, (1 << 28) // (new * c["hq"])))
        c.update(requests=1, lo=new, hi=new, clo=most // 2, chi=most)
    elif what == "mixed":
        n = rng.randint(4, 24)
        new = _log(rng, 100, 2048)
        most = max(64, min(6000, (1 << 30) // (n * new * c["hq"])))
        c.update(requests=n, lo=0, hi=1, clo=1, chi=most, chunk=new)
    else:
        n = rng.randint(1, 6)
        new = int(math.sqrt((1 << 31) / (n * c["hq"])))
        new = _log(rng, 64, min(4096, new))
        c.update(requests=n, lo=max(1, new // 3), hi=new, clo=0, chi=0)
    return c


# ---------------------------------------------------------------------------------------------- lengths
def _lengths(case):
    """(tokens that are in the cache already, new tokens) of every request: they belong to the case."""
    rng = random.Random(case["shape"])
    n = case["requests"]
    if case["kind"] == "tables":
        return [rng.randint(0, case["context"]) for _ in range(n)], [rng.randint(case["lo"], case["hi"]) for _ in range(n)]
    new = [rng.randint(case["lo"], case["hi"]) for _ in range(n)]
    have = [rng.randint(min(case["clo"], case["chi"]), case["chi"]) for _ in range(n)]
    if case["chunk"]:
        new[rng.randrange(n)] = case["chunk"]
    return have, new


def _pages(n, page):
    return (n + page - 1) // page


# ---------------------------------------------------------------------------------------------- preparation
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def ints(v, dt=torch.int32):
        return torch.tensor(v, dtype=dt, device="cuda")

    def rnd(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).to(_DTYPES[case["dtype"]])

    s = dict(case=case)
    if kind == "verify":
        b, k, v = case["requests"], case["drafts"], case["vocab"]
        draft = torch.softmax(2 * torch.randn(b, k, v, device="cuda", generator=g), -1)  # a draft model and a target that is like it
        noise = torch.randn(b, k + 1, v, device="cuda", generator=g)
        s["target"] = torch.softmax(torch.cat([draft, draft[:, :1]], 1).log() + 0.5 * noise, -1)
        s["draft"] = draft
        s["tokens"] = torch.multinomial(draft.view(b * k, v), 1, generator=g).view(b, k)
        s["lens"] = torch.randint(0, k + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
        s["lens"][::2] = k
        s["accept"] = torch.rand(b, k, device="cuda", generator=g)
        s["sample"] = torch.rand(b, device="cuda", generator=g)
        return s
    page = case["page"]
    if kind == "append":
        t, hq, hkv = case["tokens"], case["hq"], case["hkv"]
        pages = _pages(t, page) + 3
        s["qkv"] = rnd(t + case["pad"], (hq + 2 * hkv) * _D)
        s["k"], s["v"] = rnd(pages, hkv, page, _D), rnd(pages, hkv, page, _D)
        s["slots"] = torch.full((t + case["pad"],), -1, dtype=torch.int64, device="cuda")
        s["slots"][:t] = torch.randperm(pages * page, device="cuda", generator=g)[:t]
        s["positions"] = torch.randint(0, case["context"], (t + case["pad"],), device="cuda", generator=g, dtype=torch.int32)
        return s
    have, new = _lengths(case)
    total = [a + b for a, b in zip(have, new)]
    width = max(1, max(_pages(n, page) for n in total)) + 1
    in_use = have if kind == "tables" else total
    counts = [_pages(n, page) for n in in_use]
    spare = sum(_pages(n, page) for n in total) - sum(counts) + 5
    order = torch.randperm(sum(counts) + spare, device="cuda", generator=g).to(torch.int32)
    count = ints(counts)
    first = torch.cumsum(count, 0) - count
    col = torch.arange(width, device="cuda", dtype=torch.int32)
    at = (first[:, None] + col[None]).clamp(max=order.numel() - 1)
    s["table"] = torch.where(col[None] < count[:, None], order[at.long()], torch.full_like(at, -1, dtype=torch.int32))
    if kind == "tables":
        s["lens"], s["new"], s["keep"] = ints(have), ints(new), ints(have)
        s["free"] = order[sum(counts):].clone()
        s["n_free"] = ints([spare])
        s["rows"] = sum(new) + 3
        return s
    hq, hkv = case["hq"], case["hkv"]
    s["k"], s["v"] = rnd(order.numel(), hkv, page, _D), rnd(order.numel(), hkv, page, _D)
    s["lens"] = ints(total)
    s["cu_new"] = torch.cat([ints([0]), torch.cumsum(ints(new), 0).to(torch.int32)])
    s["q"] = rnd(max(1, sum(new)), hq * _D)
    s["max_new"], s["max_len"] = max(1, max(new)), max(total)
    return s


# ---------------------------------------------------------------------------------------------- one pass, plain
def _extend(table, lens, new, free, n_free, page, rows):
    old, after = (lens + page - 1) // page, (lens + new + page - 1) // page
    need = after - old
    first = torch.cumsum(need, 0) - need
    lack = (need.sum() > n_free[0]).int()
    long = (lens + new > table.shape[1] * page).any().int()
    many = (new.sum() > rows).int()
    less = (new < 0).any().int()
    status = (lack + 2 * long + 4 * many + 8 * less).view(1).to(torch.int32)
    ok = status[0] == 0
    col = torch.arange(table.shape[1], device=table.device)[None]
    k = first[:, None] + col - old[:, None]
    fresh = (col >= old[:, None]) & (col < after[:, None]) & ok
    table.copy_(torch.where(fresh, free[(n_free[0] - 1 - k).clamp(0, free.numel() - 1).long()], table))
    took = torch.where(ok, new, torch.zeros_like(new))
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(took, 0).to(torch.int32)])
    t = torch.arange(rows, device=table.device, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], t, right=True).clamp(max=lens.numel() - 1)
    live = t < cu[-1]
    pos = torch.where(live, lens[seq] + t - cu[seq], torch.zeros_like(t))
    slots = table[seq, (pos // page).long()].long() * page + pos % page
    slots = torch.where(live, slots, torch.full_like(slots, -1))
    lens.add_(took)
    n_free.sub_(torch.where(ok, need.sum(), torch.zeros_like(need.sum())).to(torch.int32))
    return cu, slots, pos, status


def _trim(table, lens, keep, free, n_free, page):
    old, after = (lens + page - 1) // page, (keep + page - 1) // page
    drop = old - after
    first = torch.cumsum(drop, 0) - drop
    full = (n_free[0] + drop.sum() > free.numel()).int()
    bad = ((keep > lens) | (keep < 0)).any().int()
    status = (full + 2 * bad).view(1).to(torch.int32)
    ok = status[0] == 0
    col = torch.arange(table.shape[1], device=table.device)[None]
    gone = (col >= after[:, None]) & (col < old[:, None]) & ok
    at = n_free[0] + drop.sum() - 1 - (first[:, None] + col - after[:, None])
    room = torch.cat([free, free[:1]])  # its last place takes what stays
    room[torch.where(gone, at, torch.full_like(at, free.numel())).long()] = table
    free.copy_(room[:-1])
    table.copy_(torch.where(gone, torch.full_like(table, -1), table))
    lens.copy_(torch.where(ok, keep, lens))
    n_free.add_(torch.where(ok, drop.sum(), torch.zeros_like(drop.sum())).to(torch.int32))
    return status


def _append(qkv, k, v, slots, positions, hq, hkv):
    half = _D // 2
    inv = _THETA ** (-torch.arange(half, device=qkv.device, dtype=torch.float64) / half)
    angle = positions.double()[:, None] * inv[None]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = qkv.view(qkv.shape[0], hq + 2 * hkv, _D)
    a, b = x[:, :hq + hkv, :half].float(), x[:, :hq + hkv, half:].float()
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(qkv.dtype)
    live = slots >= 0
    page = k.shape[2]
    # rows without a slot write what stands there already
    at, off = (slots.clamp(0) // page)[live], (slots % page)[live]
    k[at, :, off] = y[:, hq:][live]
    v[at, :, off] = x[:, hq + hkv:][live]
    return y[:, :hq].reshape(qkv.shape[0], hq * _D)


def _attention(q, k, v, table, lens, cu_new, hq, hkv, max_new, max_len):
    n, page, group = lens.numel(), k.shape[2], hq // hkv
    at = table[:, :_pages(max_len, page)].clamp(0).long()
    keys = k[at].permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, _D).float()      # [request, KV head, position, dimension]
    vals = v[at].permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, _D).float()
    new = cu_new[1:] - cu_new[:-1]
    j = torch.arange(max_new, device=q.device)
    live = j[None] < new[:, None]
    rows = (cu_new[:-1, None] + j[None]).clamp(max=q.shape[0] - 1).long()
    qs = q.view(-1, hkv, group, _D)[rows].permute(0, 2, 3, 1, 4).reshape(n, hkv, group * max_new, _D).float()
    limit = (lens - new)[:, None] + j[None] + 1                              # positions that a token sees
    p = torch.arange(keys.shape[2], device=q.device)
    seen = (p[None, None] < limit[:, :, None])[:, None, None].expand(n, 1, group, max_new, -1).reshape(n, 1, group * max_new, -1)
    scores = (qs @ keys.transpose(2, 3)).mul_(1 / math.sqrt(_D)).masked_fill_(~seen, float("-inf"))
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    o = (scores @ vals).div_(scores.sum(-1, keepdim=True))
    o = o.view(n, hkv, group, max_new, _D).permute(0, 3, 1, 2, 4).reshape(n, max_new, hq * _D).to(q.dtype)
    out = torch.zeros_like(q)
    out[rows[live]] = o[live]
    return out


def _verify(target, draft, tokens, lens, accept, sample):
    b, k = tokens.shape
    p = target[:, :k].gather(2, tokens[..., None])[..., 0].double()
    q = draft.gather(2, tokens[..., None])[..., 0].double()
    j = torch.arange(k, device=tokens.device)[None]
    good = (accept.double() * q < p) & (j < lens[:, None])
    n = torch.cumprod(good.int(), 1).sum(1)                                  # accepted
    row = torch.arange(b, device=tokens.device)
    at = target[row, n].double()
    left = (at - draft[row, n.clamp(max=k - 1)].double()).clamp(min=0)
    use = ((n < lens) & (left.sum(-1) > 0))[:, None]
    weight = torch.where(use, left, at)
    cdf = torch.cumsum(weight, -1)
    word = (cdf > sample.double()[:, None] * cdf[:, -1:]).int().argmax(-1)
    i = torch.arange(k + 1, device=tokens.device)[None]
    wide = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(i < n[:, None], wide, torch.where(i == n[:, None], word[:, None], torch.full_like(wide, -1)))
    return out, n.to(torch.int32)


# ---------------------------------------------------------------------------------------------- one pass
_workspace = {}


def _attention_workspace(s):
    """The scratch of a program that calls the attention: made once, for its largest call."""
    from gpu_ipc_example_b200._ext import load

    c = s["case"]
    need = load().paged_attention_workspace_bytes(c["hq"] // c["hkv"], s["max_new"], torch.cuda.current_device())
    if "ws" not in _workspace or _workspace["ws"].numel() < need:
        _workspace["ws"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
    return _workspace["ws"]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        from gpu_ipc_example_b200._ext import load

        load()
        ops = torch.ops.b200ipc
        if kind == "tables":
            cu, slots, pos, status = ops.paged_extend(s["table"], s["lens"], s["new"], s["free"], s["n_free"], c["page"], s["rows"])
            status2 = ops.paged_trim(s["table"], s["lens"], s["keep"], s["free"], s["n_free"], c["page"])
            return cu, slots, pos, status, status2, s["table"], s["lens"], s["free"], s["n_free"]
        if kind == "append":
            q = ops.rope_paged_append(s["qkv"], s["k"], s["v"], s["slots"], s["positions"], c["hq"], c["hkv"], _THETA)
            return q, s["k"], s["v"]
        if kind == "attention":
            return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu_new"], _attention_workspace(s), c["hq"], c["hkv"],
                                       s["max_new"])
        return ops.verify_drafts(s["target"], s["draft"], s["tokens"], s["lens"], s["accept"], s["sample"])
    if kind == "tables":
        cu, slots, pos, status = _extend(s["table"], s["lens"], s["new"], s["free"], s["n_free"], c["page"], s["rows"])
        status2 = _trim(s["table"], s["lens"], s["keep"], s["free"], s["n_free"], c["page"])
        return cu, slots, pos, status, status2, s["table"], s["lens"], s["free"], s["n_free"]
    if kind == "append":
        return _append(s["qkv"], s["k"], s["v"], s["slots"], s["positions"], c["hq"], c["hkv"]), s["k"], s["v"]
    if kind == "attention":
        return _attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu_new"], c["hq"], c["hkv"], s["max_new"], s["max_len"])
    return _verify(s["target"], s["draft"], s["tokens"], s["lens"], s["accept"], s["sample"])


# ---------------------------------------------------------------------------------------------- what it costs at least
def work(case):
    kind = case["kind"]
    if kind == "verify":
        # a row of the target's probabilities and one of the drafts' for each request, and what is looked up
        return {"bytes": case["requests"] * (8 * case["vocab"] + case["drafts"] * 28 + 20), "flops": 3 * case["requests"] * case["vocab"]}
    if kind == "append":
        heads, t = case["hq"] + 2 * case["hkv"], case["tokens"]
        pad = case["pad"] * case["hq"] * _D * 2 * 2
        return {"bytes": t * (2 * heads * _D * 2 + 12) + pad, "flops": t * (case["hq"] + case["hkv"]) * 3 * _D}
    have, new = _lengths(case)
    if kind == "tables":
        page = case["page"]
        taken = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(have, new))
        # lengths in and out twice, slots and positions out, the new pages from the list into the table and back
        return {"bytes": case["requests"] * 28 + (sum(new) + 3) * 12 + taken * 16, "flops": case["requests"] * 8 + sum(new) * 4}
    hq, hkv = case["hq"], case["hkv"]
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(have, new))
    cached = sum(a + b for a, b in zip(have, new) if b)
    return {"bytes": cached * hkv * _D * 2 * 2 + 2 * sum(new) * hq * _D * 2, "flops": 4 * pairs * hq * _D}


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    kind = case["kind"]
    if kind in ("tables", "verify"):
        return None  # whole numbers
    s = prepare(case, seed)
    if kind == "append":
        hq, hkv, page = case["hq"], case["hkv"], case["page"]
        x = s["qkv"].double().unflatten(1, (hq + 2 * hkv, _D))
        freq = torch.exp(torch.arange(_D // 2, device="cuda", dtype=torch.float64) * (-2 * math.log(_THETA) / _D))
        turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), torch.outer(s["positions"].double(), freq))[:, None]
        z = torch.complex(x[:, :hq + hkv, :_D // 2].contiguous(), x[:, :hq + hkv, _D // 2:].contiguous()) * turn
        y = torch.cat([z.real, z.imag], -1)
        k, v = s["k"].double(), s["v"].double()
        for t in range(0, case["tokens"]):
            if t % 512:
                continue
            part = s["slots"][t:min(t + 512, case["tokens"])]
            rows = slice(t, t + part.numel())
            k[part // page, :, part % page] = y[rows, hq:]
            v[part // page, :, part % page] = x[rows, hq + hkv:]
        return y[:, :hq].flatten(1), k, v
    hq, hkv, page, group = case["hq"], case["hkv"], case["page"], case["hq"] // case["hkv"]
    have, new = _lengths(case)
    if 4 * sum(b * (a + b) for a, b in zip(have, new)) * hq * _D > 2e13:
        return None
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    start = 0
    for i, (a, b) in enumerate(zip(have, new)):
        pages = s["table"][i, :_pages(a + b, page)].long()
        for h in range(hkv if b else 0):
            key = s["k"][pages, h].reshape(-1, _D)[:a + b].double()
            val = s["v"][pages, h].reshape(-1, _D)[:a + b].double()
            for r in range(0, b, 512):
                e = min(r + 512, b)
                qs = s["q"][start + r:start + e].unflatten(1, (hq, _D))[:, h * group:(h + 1) * group].double()
                w = torch.einsum("tgd,pd->tgp", qs, key[:a + e]) / math.sqrt(_D)
                behind = torch.arange(a + e, device="cuda")[None, :] > torch.arange(a + r, a + e, device="cuda")[:, None]
                w = torch.softmax(w.masked_fill(behind[:, None], -math.inf), -1)
                got = torch.einsum("tgp,pd->tgd", w, val[:a + e])
                out[start + r:start + e, h * group * _D:(h + 1) * group * _D] = got.flatten(1)
        start += b
    return out
