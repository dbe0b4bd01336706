"""The operators of paged serving against the same written out in 64 bits (tests/paged_reference.py)."""
import random

import pytest
import torch

import paged_reference as ref
from gpu_ipc_example_b200._ext import load

pytestmark = pytest.mark.gpu
D = 128


def ints(v, dt=torch.int32):
    return torch.tensor(v, dtype=dt, device="cuda")


def ops():
    load()
    return torch.ops.b200ipc


# ---------------------------------------------------------------------------------------------- block tables
def make_table(rng, lens, width, page, spare):
    counts = [ref.pages_of(n, page) for n in lens]
    order = list(range(sum(counts) + spare))
    rng.shuffle(order)
    table, at = [], 0
    for c in counts:
        table.append(order[at:at + c] + [-1] * (width - c))
        at += c
    return table, order[at:]


def check_extend(lens, new, width, page, spare, rows, room=0, seed=0):
    table, free = make_table(random.Random(seed), lens, width, page, spare)
    n_free = len(free)
    free = free + [-7] * room
    want = ref.extend(table, lens, new, free, n_free, page, rows)
    t, l, f, n = ints(table), ints(lens), ints(free), ints([n_free])
    cu, slots, positions, status = ops().paged_extend(t, l, ints(new), f, n, page, rows)
    assert (t.tolist(), l.tolist(), int(n), cu.tolist(), slots.tolist(), positions.tolist(), int(status)) == want
    assert f.tolist() == free
    return (t, l, f, n), (table, lens, free, n_free), want


@pytest.mark.parametrize("requests,page,hi,context", [(1, 64, 1, 0), (1, 16, 300, 33), (3, 1, 5, 7), (32, 64, 1, 2048), (33, 48, 17, 500), (513, 16, 9, 300),
                                                      (700, 32, 0, 100), (1025, 128, 3, 900), (100, 16, 100, 5000), (8192, 16, 2, 40)])
def test_extend_and_trim_are_inverse(requests, page, hi, context):
    rng = random.Random(requests)
    lens = [rng.randint(0, context) for _ in range(requests)]
    new = [rng.choice([0, hi, rng.randint(0, hi)]) for _ in range(requests)]
    width = max(1, max(ref.pages_of(a + b, page) for a, b in zip(lens, new)))
    need = sum(ref.pages_of(a + b, page) - ref.pages_of(a, page) for a, b in zip(lens, new))
    own = sum(ref.pages_of(a, page) for a in lens)  # pages that were taken before
    (t, l, f, n), before, want = check_extend(lens, new, width, page, need, sum(new) + 2, room=own)
    assert want[6] == 0 and int(n) == 0

    def trim(keep):
        want = ref.trim(t.tolist(), l.tolist(), keep, f.tolist(), int(n), page)
        status = ops().paged_trim(t, l, ints(keep), f, n, page)
        assert (t.tolist(), l.tolist(), f.tolist(), int(n), int(status)) == want and want[4] == 0

    trim(lens)  # in one go: what was there before
    assert (t.tolist(), l.tolist(), f.tolist(), int(n)) == before
    assert ops().paged_extend(t, l, ints(new), f, n, page, sum(new))[3].item() == 0
    trim([a + rng.randint(0, b) for a, b in zip(lens, new)])  # drafts that were turned down
    trim([0] * requests)                                      # all requests are done
    assert sorted(f.tolist()) == list(range(need + own))


@pytest.mark.parametrize("lens,new,width,spare,rows,status", [
    ([10, 20], [30, 40], 8, 3, 70, 1),    # four pages wanted, three there
    ([10, 20], [30, 40], 4, 9, 69, 4),    # a row too few
    ([10, 120], [30, 9], 8, 9, 70, 2),    # 129 tokens in a row of 128
    ([10, 20], [30, -1], 8, 9, 70, 8),
    ([10, 20, 127], [30, 40, 2], 8, 3, 60, 7),
    ([10, 20], [2 ** 31 - 1, 2 ** 31 - 1], 8, 9, 70, 2),
])
def test_extend_that_cannot_be_changes_nothing(lens, new, width, spare, rows, status):
    state, before, want = check_extend(lens, new, width, 16, spare, rows, room=2)
    assert want[6] == status
    assert (state[0].tolist(), state[1].tolist(), state[2].tolist(), int(state[3])) == before


def test_extend_beyond_what_an_int_counts_changes_nothing():
    """Pages so large that a row of the table holds more than 2^31 tokens."""
    for len_, new, status in ((2 ** 31 - 2, 2, 2), (2 ** 31 - 3, 2, 0)):
        t, l, n = ints([[0] * 2048 + [-1] * 8]), ints([len_]), ints([4])
        cu, slots, positions, said = ops().paged_extend(t, l, ints([new]), ints([9, 8, 7, 6]), n, 1 << 20, 3)
        assert (int(said), int(l), int(n)) == (status, len_ if status else len_ + new, 4)
        assert positions.tolist() == ([0, 0, 0] if status else [len_, len_ + 1, 0]) and cu.tolist() == [0, 0 if status else 2]


def test_trim_that_cannot_be_changes_nothing():
    table, free = make_table(random.Random(1), [40, 50], 4, 16, 3)
    for keep, n_free, status in (([41, 0], 3, 2), ([3, -1], 3, 8), ([0, 0], 1, 1), ([0, 0], -1, 1)):
        room = free + [-7] * (0 if status == 1 else 9)
        t, l, f, n = ints(table), ints([40, 50]), ints(room), ints([n_free])
        assert int(ops().paged_trim(t, l, ints(keep), f, n, 16)) == status
        assert (t.tolist(), l.tolist(), f.tolist(), int(n)) == (table, [40, 50], room, n_free)


# ---------------------------------------------------------------------------------------------- rotary positions and append
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,hq,hkv,page,extra", [(1, 8, 1, 64, 0), (37, 3, 3, 16, 8), (130, 20, 4, 48, 0), (5, 65, 5, 1, 64)])
def test_append(dtype, rows, hq, hkv, page, extra):
    g = torch.Generator(device="cuda").manual_seed(rows)
    wide = torch.randn(rows, (hq + 2 * hkv) * D + extra, device="cuda", generator=g).to(dtype)
    qkv = wide[:, :(hq + 2 * hkv) * D]
    pages = ref.pages_of(rows, page) + 2
    k = torch.full((pages, hkv, page, D), float("nan"), device="cuda", dtype=dtype)
    v = k.clone()
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:rows]
    slots[rows // 2] = -1          # rows without a place in the cache
    if rows > 4:
        slots[3] = pages * page
        slots[4] = -(2 ** 40)
    positions = torch.randint(0, 130000, (rows,), device="cuda", generator=g, dtype=torch.int32)
    positions[0] = 0
    keep = wide.clone()
    q = ops().rope_paged_append(qkv, k, v, slots, positions, hq, hkv, 5e5)
    assert torch.equal(wide, keep)
    x = qkv.cpu().double().view(rows, hq + 2 * hkv, D)
    y = ref.rotate(x[:, :hq + hkv], positions.cpu(), 5e5)
    # one rounding of half a step at the end; sine, cosine and two products in fp32: 2^-21 of the pair's length
    tol = lambda z, w: torch.finfo(dtype).eps / 2 * z.abs() + 2.0 ** -21 * w + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    size = x[:, :hq + hkv].abs()
    size = size + size.roll(D // 2, -1)
    assert ((q.cpu().double().view(rows, hq, D) - y[:, :hq]).abs() <= tol(y[:, :hq], size[:, :hq])).all()
    kk, vv = k.cpu().double(), v.cpu().double()
    told = set()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            told.add(s)
            assert ((kk[s // page, :, s % page] - y[t, hq:]).abs() <= tol(y[t, hq:], size[t, hq:])).all()
            assert torch.equal(vv[s // page, :, s % page], x[t, hq + hkv:])
    rest = torch.tensor([s for s in range(pages * page) if s not in told])
    for c in (kk, vv):
        assert c[rest // page, :, rest % page].isnan().all()  # nothing else is written


def test_append_of_no_rows():
    k = torch.zeros(2, 1, 16, D, device="cuda", dtype=torch.float16)
    q = ops().rope_paged_append(torch.empty(0, 3 * D, device="cuda", dtype=torch.float16), k, k.clone(), ints([], torch.int64), ints([]), 1, 1, 1e4)
    assert q.shape == (0, D)


# ---------------------------------------------------------------------------------------------- attention
def paged_problem(dtype, page, hq, hkv, have, new, seed=0, behind=0, scale=1.0, extra=0):
    """Everything that is not a token of some request is NaN: the rest of the pages, and pages of nobody."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = [a + b for a, b in zip(have, new)]
    width = max(1, max(ref.pages_of(n, page) for n in total)) + 1
    table, free = make_table(random.Random(seed), total, width, page, 3)
    pages = sum(len([x for x in r if x >= 0]) for r in table) + len(free)
    k = torch.full((pages, hkv, page, D), float("nan"), device="cuda", dtype=dtype)
    v = torch.full_like(k, float("inf"))
    for i, n in enumerate(total):
        for c in range(ref.pages_of(n, page)):
            m = min(page, n - c * page)
            k[table[i][c], :, :m] = (torch.randn(hkv, m, D, device="cuda", generator=g)).to(dtype)
            v[table[i][c], :, :m] = (torch.randn(hkv, m, D, device="cuda", generator=g)).to(dtype)
    cu = [0]
    for b in new:
        cu.append(cu[-1] + b)
    q = (scale * torch.randn(cu[-1] + behind, hq * D + extra, device="cuda", generator=g)).to(dtype)
    return q, k, v, table, total, cu


def workspace(hq, hkv, max_new):
    n = load().paged_attention_workspace_bytes(hq // hkv, max_new, torch.cuda.current_device())
    return torch.zeros(n, dtype=torch.uint8, device="cuda")


def attend(p, hq, hkv, max_new=None, ws=None):
    q, k, v, table, total, cu = p
    max_new = max_new or max(1, max(b - a for a, b in zip(cu, cu[1:])))
    ws = workspace(hq, hkv, max_new) if ws is None else ws
    out = ops().paged_attention(q, k, v, ints(table), ints(total), ints(cu), ws, hq, hkv, max_new)
    assert int(ws[:4].view(torch.int32)) == 0  # no wait gave up
    return out


def assert_attention(out, p, hq, hkv):
    q, k, v, table, total, cu = p
    want, mag = ref.attention(q, torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0), table, total, cu, hq, hkv)
    eps = torch.finfo(q.dtype).eps
    # One rounding of the result and one of every weight, half a step each (of the result, of the weighted sum of |v|); scores and sums in
    # fp32 are good to 2^-14 of the weight.  Weights below the normal range of fp16 are off by 2^-25 of the largest one.
    lost = max(total) * 2.0 ** -25 * 6 if q.dtype == torch.float16 else 0.0
    tol = eps / 2 * want.abs() * 1.01 + (eps / 2 + 2.0 ** -14) * mag + lost
    off = (out.cpu().double() - want).abs()
    assert torch.isfinite(out).all()
    assert (off <= tol).all(), float((off / tol.clamp(min=1e-30)).max())
    assert (out[cu[-1]:] == 0).all()  # rows behind the last request


SHAPES = [  # hq, hkv, page, have, new
    (8, 1, 16, [0], [1]),
    (8, 1, 64, [299], [1]),
    (8, 8, 16, [15, 16, 17, 0], [1, 1, 1, 1]),
    (5, 1, 32, [31, 63, 64, 2000], [1, 0, 1, 1]),
    (16, 2, 128, [127, 128, 129, 1000], [1, 1, 2, 3]),
    (16, 2, 32, [0, 500, 33], [5, 5, 5]),
    (6, 2, 64, [10, 0, 700], [11, 7, 13]),
    (8, 4, 16, [100] * 40, [1] * 40),
    (8, 1, 64, [4000, 1], [1, 1]),
    (32, 1, 64, [70, 130], [2, 2]),
    (64, 1, 16, [5, 100], [1, 3]),
    (8, 1, 64, [0], [16]),
    (8, 1, 16, [0, 40], [17, 33]),
    (8, 1, 128, [300], [64]),
    (4, 2, 32, [0], [257]),
    (8, 2, 64, [1000, 0, 5], [129, 200, 1]),
    (5, 5, 16, [77], [300]),
    (7, 1, 64, [0, 0], [100, 1]),
    (12, 4, 128, [2047], [130]),
    (1, 1, 32, [129, 0, 0, 1], [128, 127, 0, 129]),
    (3, 1, 64, [5000], [200]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,page,have,new", SHAPES)
def test_attention(dtype, hq, hkv, page, have, new):
    p = paged_problem(dtype, page, hq, hkv, have, new, seed=len(have) + hq)
    assert_attention(attend(p, hq, hkv), p, hq, hkv)


@pytest.mark.parametrize("new", [[1, 2, 1], [90, 1, 0]])
def test_attention_of_a_padded_batch_in_wider_rows(new):
    """q is the front of the projection's rows, rows stand behind the last request, and max_new is only a bound."""
    hq, hkv = 8, 2
    p = paged_problem(torch.float16, 64, hq, hkv, [70, 0, 300], new, behind=13, extra=2 * hkv * D)
    q = p[0][:, :hq * D]
    assert_attention(attend((q,) + p[1:], hq, hkv, max_new=200), (q,) + p[1:], hq, hkv)


@pytest.mark.parametrize("new", [[3, 2], [100, 90]])
def test_attention_of_tokens_that_see_nothing(new):
    """A request whose length is less than its new tokens: the first rows have no position to look at."""
    hq, hkv = 8, 1
    q, k, v, table, total, cu = paged_problem(torch.bfloat16, 16, hq, hkv, [50, 60], new)
    p = (q, k, v, table, [1, total[1]], cu)
    out = attend(p, hq, hkv)
    assert (out[:new[0] - 1] == 0).all() and float(out[new[0] - 1].abs().max()) > 0
    assert_attention(out, p, hq, hkv)
    p = (q, k, v, table, [0, total[1]], cu)
    assert_attention(attend(p, hq, hkv), p, hq, hkv)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 150])
def test_attention_of_steep_scores(dtype, new):
    """Scores of some hundred: one position takes everything, and the running maximum jumps."""
    hq, hkv = 8, 2
    p = paged_problem(dtype, 64, hq, hkv, [900, 20], [new, new], scale=40.0)
    assert_attention(attend(p, hq, hkv), p, hq, hkv)


@pytest.mark.parametrize("requests,new", [(300, 2), (1000, 2), (1300, 20), (2500, 1)])
def test_attention_of_a_batch_larger_than_the_grid(requests, new):
    """More requests than CTAs, and than the threads that look through them."""
    hq, hkv = 8, 4
    rng = random.Random(requests)
    p = paged_problem(torch.float16, 16, hq, hkv, [rng.randint(0, 60) for _ in range(requests)], [rng.choice([0, rng.randint(0, new)]) for _ in range(requests)])
    assert_attention(attend(p, hq, hkv, max_new=new), p, hq, hkv)


def test_attention_gives_the_same_bits_again():
    for new in ([1, 1, 4], [200, 1, 150]):
        hq, hkv = 16, 2
        p = paged_problem(torch.float16, 64, hq, hkv, [3000, 10, 2000], new)
        first = attend(p, hq, hkv)
        assert all(torch.equal(first, attend(p, hq, hkv)) for _ in range(5))


def test_attention_call_behind_call():
    """Calls of all sorts without a pause, a workspace for all of them: every one its own result, no wait that gives up."""
    sorts = [(8, 1, 64, [700, 20, 3000], [5, 3, 8]), (16, 2, 32, [0, 900], [20, 9]), (8, 2, 64, [1000, 0, 5], [129, 200, 1]), (8, 1, 16, [400] * 5, [1] * 5),
             (32, 8, 128, [100, 0, 2000], [1, 700, 1]), (16, 2, 32, [3000] * 20, [5] * 20)]
    problems = [paged_problem(torch.bfloat16, page, hq, hkv, have, new) for hq, hkv, page, have, new in sorts]
    ws = workspace(8, 1, 700)
    args = [(q, k, v, ints(t), ints(n), ints(cu), ws, hq, hkv, max(new)) for (q, k, v, t, n, cu), (hq, hkv, _, _, new) in zip(problems, sorts)]
    outs = [None] * len(sorts)
    for rep in range(60):
        for i, a in enumerate(args):
            outs[i] = ops().paged_attention(*a)
        assert int(ws[:4].view(torch.int32)) == 0
    for out, p, (hq, hkv, *_) in zip(outs, problems, sorts):
        assert_attention(out, p, hq, hkv)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("have,new", [(0, 2), (0, 64), (100, 150), (0, 300)])
def test_later_tokens_have_no_weight_at_all(dtype, have, new):
    """The greatest values that there are behind a row's own position leave its zeros as they are."""
    hq, hkv, page = 8, 1, 64
    q, k, v, table, total, cu = paged_problem(dtype, page, hq, hkv, [have], [new], seed=new)
    half = have + new // 2
    flat = torch.zeros(total[0], hkv, D, device="cuda", dtype=dtype)
    flat[half:] = torch.finfo(dtype).max / 2
    for c in range(ref.pages_of(total[0], page)):
        m = min(page, total[0] - c * page)
        v[table[0][c], :, :m] = flat[c * page:c * page + m].transpose(0, 1)
    out = attend((q, k, v, table, total, cu), hq, hkv)
    # Rows that see such values are not asked for more than their sign: before they are divided by the sum of the weights, outputs are sums of n
    # weights of up to 2^8 times 2^127 in bf16, where fp32 ends at 2^128.
    assert (out[:new // 2] == 0).all() and (out[new // 2:] > 0).all()


def test_two_captured_graphs_share_a_workspace():
    """One of single tokens and one of chunks, replayed in turn with lengths that change between the replays."""
    hq, hkv = 8, 2
    sorts = [([500, 900], [1, 1]), ([300, 2000], [100, 60])]
    problems = [paged_problem(torch.bfloat16, 32, hq, hkv, have, new, seed=3) for have, new in sorts]
    ws = workspace(hq, hkv, 100)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs, lens = [], [], []
    with torch.cuda.stream(stream):
        for (q, k, v, table, total, cu), (_, new) in zip(problems, sorts):
            args = [q, k, v, ints(table), ints(total), ints(cu), ws, hq, hkv, max(new)]
            ops().paged_attention(*args)
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                outs.append(ops().paged_attention(*args))
            lens.append(args[4])
            outs.append(args)  # alive while the graphs are
        for less in (0, 37, 0):
            for g, n, (_, _, _, _, total, _) in zip(graphs, lens, problems):
                n.copy_(ints([t - less for t in total]))
                g.replay()
            for out, (q, k, v, table, total, cu) in zip(outs[::2], problems):
                p = (q, k, v, table, [t - less for t in total], cu)
                assert_attention(out, p, hq, hkv)
        assert int(ws[:4].view(torch.int32)) == 0
    torch.cuda.synchronize()


def test_attention_of_bad_pages_leaves_the_others_alone():
    """Pages that the cache does not have: those requests get something finite or not, the others what they should."""
    for new in ([1, 1, 1], [100, 100, 100]):
        hq, hkv = 8, 1
        q, k, v, table, total, cu = paged_problem(torch.float16, 32, hq, hkv, [70, 300, 40], new)
        bad = [list(r) for r in table]
        bad[1][0], bad[1][2], bad[1][4] = -1, k.shape[0], 2 ** 31 - 1
        out = attend((q, k, v, bad, total, cu), hq, hkv)
        torch.cuda.synchronize()
        out[cu[1]:cu[2]] = 0
        want, _ = ref.attention(q, torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0), table, total, cu, hq, hkv)
        want[cu[1]:cu[2]] = 0
        assert (out.cpu().double() - want).abs().max() < 0.01


@pytest.mark.parametrize("new,later", [(1, 1), (3, 2), (150, 70)])
def test_attention_captured_and_replayed_with_other_lengths(new, later):
    """Lengths are read on the GPU: one graph serves every step, another stream's too."""
    hq, hkv, page = 8, 2, 16
    a = paged_problem(torch.float16, page, hq, hkv, [500, 3, 100], [new] * 3, seed=1)
    b = paged_problem(torch.float16, page, hq, hkv, [20, 400, 0], [later] * 3, seed=2)
    width = max(len(a[3][0]), len(b[3][0]))
    pages = max(a[1].shape[0], b[1].shape[0])
    q = torch.zeros(3 * max(new, later), hq * D, device="cuda", dtype=torch.float16)
    k, v = (torch.zeros(pages, hkv, page, D, device="cuda", dtype=torch.float16) for _ in range(2))
    table, lens, cu = ints([[-1] * width] * 3), ints([0] * 3), ints([0] * 4)

    def fill(p):
        q.zero_()
        q[:p[0].shape[0]].copy_(p[0])
        k[:p[1].shape[0]].copy_(p[1])
        v[:p[2].shape[0]].copy_(p[2])
        table.copy_(ints([r + [-1] * (width - len(r)) for r in p[3]]))
        lens.copy_(ints(p[4]))
        cu.copy_(ints(p[5]))

    ws = workspace(hq, hkv, max(new, later))
    stream = torch.cuda.Stream()
    call = lambda: ops().paged_attention(q, k, v, table, lens, cu, ws, hq, hkv, max(new, later))
    fill(a)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
    for p in (a, b, a):
        fill(p)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        rows = p[0].shape[0]
        assert_attention(out[:rows], p, hq, hkv)
        assert (out[rows:] == 0).all()


def test_a_cache_of_more_than_two_to_the_31_elements():
    """Append to the last pages of caches of 4.5 GB each, and attention over them: short requests and long ones."""
    hq, hkv, page = 8, 2, 64
    pages = (1 << 31) // (hkv * page * D) + 2000
    k, v = (torch.empty(pages, hkv, page, D, device="cuda", dtype=torch.float16) for _ in range(2))
    for new in ([1, 2], [40, 3]):
        have = [500, 70]
        q, ks, vs, table, total, cu = paged_problem(torch.float16, page, hq, hkv, have, new)
        offset = pages - ks.shape[0]
        k[offset:].copy_(ks)
        v[offset:].copy_(vs)
        far = [[x + offset if x >= 0 else x for x in r] for r in table]
        out = attend((q, k, v, far, total, cu), hq, hkv)
        assert_attention(out, (q, ks, vs, table, total, cu), hq, hkv)
    qkv = torch.randn(3, (hq + 2 * hkv) * D, device="cuda").half()
    slots = torch.tensor([pages * page - 1, pages * page - 777, pages * page], device="cuda")  # the last one is behind the cache
    ops().rope_paged_append(qkv, k, v, slots, ints([0, 0, 0]), hq, hkv, 1e4)
    x = qkv.view(3, hq + 2 * hkv, D)
    for t, s in ((0, pages * page - 1), (1, pages * page - 777)):
        assert torch.equal(k[s // page, :, s % page], x[t, hq:hq + hkv]) and torch.equal(v[s // page, :, s % page], x[t, hq + hkv:])


def test_calls_on_another_stream_than_the_tensors():
    """Each operator runs on the current stream, whichever that is."""
    hq, hkv = 8, 2
    stream = torch.cuda.Stream()
    for new in ([1, 1], [60, 9]):
        p = paged_problem(torch.bfloat16, 32, hq, hkv, [300, 77], new)
        ws = workspace(hq, hkv, max(new))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(2_000_000)
            q = p[0].mul(2)  # behind the pause: a call on another stream would read q before it is there
            args = (ints(p[3]), ints(p[4]), ints(p[5]))
            out = ops().paged_attention(q, p[1], p[2], *args, ws, hq, hkv, max(new))
        stream.synchronize()
        assert_attention(out, (q,) + p[1:], hq, hkv)


# ---------------------------------------------------------------------------------------------- verification
def probabilities(g, *shape, zeros=0.0):
    p = torch.softmax(2 * torch.randn(*shape, device="cuda", generator=g), -1)
    if zeros:
        p = p * (torch.rand(*shape, device="cuda", generator=g) > zeros)
    return p


@pytest.mark.parametrize("b,k,vocab,zeros", [(1, 1, 1, 0.0), (3, 4, 5, 0.5), (7, 0, 1000, 0.0), (9, 3, 1001, 0.9), (32, 4, 32000, 0.0), (5, 8, 128256, 0.3), (2, 40, 130, 0.0),
                                             (4, 33, 4096, 0.0), (2, 2, 262147, 0.0)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(b, k, vocab, zeros, certain):
    g = torch.Generator(device="cuda").manual_seed(vocab + b)
    draft = probabilities(g, b, k, vocab, zeros=zeros)
    like = torch.cat([draft, probabilities(g, b, 1, vocab)], 1)
    target = 0.7 * like + 0.3 * probabilities(g, b, k + 1, vocab, zeros=zeros)
    for seed in range(4):
        if k:
            tokens = torch.multinomial(draft.view(b * k, vocab) + 1e-9, 1, generator=g).view(b, k)
        else:
            tokens = torch.empty(b, 0, dtype=torch.int64, device="cuda")
        lens = torch.randint(0, k + 1, (b,), device="cuda", generator=g, dtype=torch.int32) if seed else None
        accept, sample = torch.rand(b, k, device="cuda", generator=g), torch.rand(b, device="cuda", generator=g)
        if seed == 2:
            accept.fill_(0)
        if seed == 3:
            sample[:] = 1.0 - 2.0 ** -24
            accept.fill_(1)
        got = ops().verify_drafts(target, None if certain else draft, tokens, lens, accept, sample)
        want = ref.verify(target.cpu(), None if certain else draft.cpu(), tokens.cpu(), None if lens is None else lens.cpu(), accept.cpu(), sample.cpu())
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_verify_of_odd_probabilities():
    """Rows of zeros, NaN, drafts that no word stands for, the same distribution on both sides, numbers out of their range."""
    nan, inf = float("nan"), float("inf")
    even = [0.25] * 4
    target = torch.tensor([[[0, 0, 0, 0.0], even], [[0.5, nan, 0.5, 0], even], [even, even], [even, even], [even, [0, 0, 1, 0.0]], [[0, 1, 0, 0.0], even],
                           [even, even], [[0.5, 0.5, 0, 0], even]], device="cuda")
    draft = torch.tensor([[even], [[0, 1, 0, 0.0]], [even], [even], [even], [[0, 1, 0, 0.0]], [[1, 0, 0, 0.0]], [[0.5, 0.5, 0, 0]]], device="cuda")
    tokens = ints([[1], [1], [-1], [4], [0], [1], [0], [2]], torch.int64)
    accept = torch.tensor([[0.0], [0.0], [0.0], [0.0], [0.5], [0.99], [0.3], [0.0]], device="cuda")
    sample = torch.tensor([0.5, 0.7, 0.6, 0.0, 0.1, 0.9, nan, 1.5], device="cuda")
    got = ops().verify_drafts(target, draft, tokens, None, accept, sample)
    want = ref.verify(target.cpu(), draft.cpu(), tokens.cpu(), None, accept.cpu(), sample.cpu())
    assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()
    assert got[0][0].tolist() == [-1, -1]  # nothing to draw from
    assert got[0][1].tolist() == [2, -1] and got[0][4].tolist() == [0, 2]


def test_verify_of_strided_and_shared_probabilities():
    g = torch.Generator(device="cuda").manual_seed(0)
    wide = probabilities(g, 6, 5, 1003)
    target = wide[:, 1:4, 1:1002]                     # unaligned rows
    draft = probabilities(g, 1, 1, 1001).expand(6, 2, 1001)  # one row for all
    tokens = torch.randint(0, 1001, (6, 2), device="cuda", generator=g)
    accept, sample = torch.rand(6, 2, device="cuda", generator=g), torch.rand(6, device="cuda", generator=g)
    got = ops().verify_drafts(target, draft, tokens, None, accept, sample)
    want = ref.verify(target.cpu(), draft.cpu(), tokens.cpu(), None, accept.cpu(), sample.cpu())
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_verified_words_have_the_target_distribution():
    """Whatever the drafts' distribution, the first word of many requests is drawn from the target's (the point of the method): counts within
    five standard deviations of the binomial's."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n, vocab = 20000, 6
    target = probabilities(g, 1, 2, vocab).expand(n, 2, vocab)
    draft = probabilities(g, 1, 1, vocab).expand(n, 1, vocab)
    tokens = torch.multinomial(draft[:, 0], 1, generator=g)
    got, _ = ops().verify_drafts(target, draft, tokens, None, torch.rand(n, 1, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g))
    counts = torch.bincount(got[:, 0], minlength=vocab).double().cpu()
    p = target[0, 0].double().cpu()
    assert ((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1).all()
