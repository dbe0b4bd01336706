"""Paged attention where infinities and NaN are in what the tokens see, verification of probabilities that are NaN, and other streams than the
tensors' own."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import D, attend, ints, ops, paged_problem

pytestmark = pytest.mark.gpu

# hq, new: up to 16 rows a request; up to 128 (two halves of every tile); more (two accumulators, and a second item)
ROWS = [(8, 1), (8, 2), (8, 5), (2, 50), (3, 50), (4, 70), (7, 20)]


def rows_that_see(cu, total, i, p):
    """Rows of request i that see position p: [cu[i] + first, cu[i + 1])."""
    new = cu[i + 1] - cu[i]
    return slice(cu[i] + max(0, p - (total[i] - new)), cu[i + 1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("keys", [1, 2])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("hq,new", ROWS)
def test_a_key_without_a_score_is_seen(dtype, keys, bad, hq, new):
    """A key of NaN, or one with a score of +inf (inf - inf in the softmax), at every place of a tile, one request each: rows that see it are NaN, the
    rows before it what they are without it."""
    page, have = 64, 130
    p = paged_problem(dtype, page, hq, 1, [have] * 128, [new] * 128, seed=hq)
    q, k, v, table, total, cu = p
    q.view(-1, hq, D)[..., 0] = 1
    clean = k.clone()
    places = [[o + 10, (o ^ (keys - 1)) + 10] for o in range(128)]  # over two tiles; the last ones are new tokens themselves
    for i, at in enumerate(places):
        for x in at:
            k[table[i][x // page], 0, x % page, 0] = float(bad)
    out = attend(p, hq, 1)
    for i, at in enumerate(places):
        see = rows_that_see(cu, total, i, min(at))
        assert out[see].isnan().all(), (i, at)
        out[see] = 0
    want, mag = ref.attention(q, torch.nan_to_num(clean, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0), table, total, cu, hq, 1)
    for i, at in enumerate(places):
        want[rows_that_see(cu, total, i, min(at))] = 0
    # as in assert_attention: half a step of the result and of every weight, 2^-14 for scores and sums, what fp16 loses of small weights
    eps = torch.finfo(dtype).eps
    tol = eps / 2 * want.abs() * 1.01 + (eps / 2 + 2.0 ** -14) * mag + (max(total) * 2.0 ** -25 * 6 if dtype == torch.float16 else 0)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("hq,new", [(8, 1), (8, 5), (4, 70)])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("place", [0, 3006, 3007, 5990])
def test_a_key_without_a_score_is_seen_through_the_join(hq, new, bad, place):
    """The same where a request is in many pieces, one of which has the key."""
    q, k, v, table, total, cu = p = paged_problem(torch.bfloat16, 64, hq, 1, [6000], [new])
    q.view(-1, hq, D)[..., 0] = 1
    k[table[0][place // 64], 0, place % 64, 0] = float(bad)
    assert attend(p, hq, 1).isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,new", ROWS)
def test_scores_of_minus_infinity(dtype, hq, new):
    """Keys with a score of -inf have no weight; where a row sees no others its softmax is 0 / 0."""
    page, lens = 32, [0, 3, 200, 64, 3000]
    q, k, v, table, total, cu = p = paged_problem(dtype, page, hq, 1, lens, [new] * 5, seed=new)
    q.view(-1, hq, D)[..., 0] = -1
    for i in (0, 1, 3, 4):
        for x in range(total[i]):
            k[table[i][x // page], 0, x % page, 0] = float("inf")
    some = list(range(0, total[2], 3))
    for x in some:
        k[table[2][x // page], 0, x % page, 0] = float("inf")
    out = attend(p, hq, 1)
    for i in (0, 1, 3, 4):
        assert out[cu[i]:cu[i + 1]].isnan().all()
    rest = [x for x in range(total[2]) if x % 3]
    kk, vv = (torch.stack([c[table[2][x // page], 0, x % page] for x in rest]).cpu().double() for c in (k, v))
    qq = q[cu[2]:cu[3]].cpu().double().view(new, hq, D)
    s = torch.einsum("thd,pd->thp", qq, kk) / D ** 0.5
    dark = torch.tensor(rest)[None] > (total[2] - new + torch.arange(new))[:, None]
    w = torch.softmax(s.masked_fill(dark[:, None], -float("inf")), -1)
    want, mag = w @ vv, w @ vv.abs()
    eps = torch.finfo(dtype).eps
    tol = eps / 2 * want.abs() * 1.01 + (eps / 2 + 2.0 ** -14) * mag + (total[2] * 2.0 ** -25 * 6 if dtype == torch.float16 else 0)
    assert ((out[cu[2]:cu[3]].cpu().double().view(new, hq, D) - want).abs() <= tol).all()


@pytest.mark.parametrize("hq,new", [(8, 2), (8, 9), (4, 70)])
def test_rows_that_see_nothing_are_zeros_whatever_the_values(hq, new):
    """A request that is shorter than its new tokens, infinities among the values of the last of them."""
    q, k, v, table, total, cu = paged_problem(torch.float16, 16, hq, 1, [0, 90], [new, new])
    v[table[0][0], :, 0] = float("inf")
    out = attend((q, k, v, table, [1, total[1]], cu), hq, 1)
    assert (out[:new - 1] == 0).all()


def test_verify_of_drafts_that_are_nan():
    """A draft whose probability is NaN is turned down, and words of NaN have no weight behind it; where none has any, the target's own."""
    nan = float("nan")
    target = torch.tensor([[[0.25, 0.5, 0.25, 0], [1, 0, 0, 0.0]], [[0.25, 0.25, 0.5, 0], [1, 0, 0, 0.0]], [[0.0, 1, 0, 0], [1, 0, 0, 0.0]]], device="cuda")
    draft = torch.tensor([[[0.5, nan, 0.1, 0.4]], [[0.1, nan, nan, 0.1]], [[nan] * 4]], device="cuda")
    tokens, accept, sample = ints([[1]] * 3, torch.int64), torch.zeros(3, 1, device="cuda"), torch.full((3,), 0.5, device="cuda")
    got = ops().verify_drafts(target, draft, tokens, None, accept, sample)
    want = ref.verify(target.cpu(), draft.cpu(), tokens.cpu(), None, accept.cpu(), sample.cpu())
    assert got[0].tolist() == want[0].tolist() == [[2, -1], [0, -1], [1, -1]] and got[1].tolist() == [0, 0, 0]


def test_tables_append_and_verify_on_another_stream():
    """What they read is made behind a pause on that stream: a call on another one would not see it."""
    stream = torch.cuda.Stream()
    lens, new, keep = ints([5, 0, 40]), ints([20, 3, 0]), ints([7, 0, 39])
    table, free, n_free = ints([[0, -1], [-1, -1], [1, 2]]), ints([9, 8, 7, 6, 5, 4]), ints([3])
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(23, 4 * D, device="cuda", generator=g).half()
    k, v = (torch.zeros(10, 1, 32, D, device="cuda", dtype=torch.float16) for _ in range(2))
    target = torch.softmax(torch.randn(3, 3, 1000, device="cuda", generator=g), -1)
    tokens, accept, sample = torch.randint(0, 1000, (3, 2), device="cuda", generator=g), torch.rand(3, 2, device="cuda", generator=g), torch.rand(3, device="cuda", generator=g)
    torch.cuda.synchronize()

    def calls():
        n, ks, vs = new + 0, k.clone(), v.clone()
        t, l, f, m = table.clone(), lens.clone(), free.clone(), n_free.clone()
        cu, slots, positions, status = ops().paged_extend(t, l, n, f, m, 32, 23)
        q = ops().rope_paged_append(x.mul(2), ks, vs, slots, positions, 2, 1, 1e4)
        words = ops().verify_drafts(target.mul(1), None, tokens, None, accept, sample)
        said = ops().paged_trim(t, l, keep, f, m, 32)
        return [cu, slots, positions, status, q, ks, vs, *words, said, t, l, f, m]

    want = [c.clone() for c in calls()]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(5_000_000)
        got = calls()
    stream.synchronize()
    assert int(want[3]) == 0 and int(want[9]) == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))
