"""The operators of paged serving written out in 64 bits (or whole numbers) on the CPU, request by request, for the tests."""
import math

import torch

D = 128


def pages_of(n, page):
    return -(-n // page)


def extend(table, lens, new, free, n_free, page, rows):
    """Lists in, lists out; nothing changes where the status is not 0."""
    status = 0
    need = 0
    for n, a in zip(lens, new):
        if n < 0 or a < 0:
            status |= 8
        elif n + a > len(table[0]) * page:
            status |= 2
        else:
            need += pages_of(n + a, page) - pages_of(n, page)
    fits = [a for n, a in zip(lens, new) if n >= 0 and a >= 0 and n + a <= len(table[0]) * page]
    if need > n_free:
        status |= 1
    if sum(fits) > rows:
        status |= 4
    table, lens = [list(r) for r in table], list(lens)
    cu, slots, positions = [0] * (len(lens) + 1), [-1] * rows, [0] * rows
    if status == 0:
        t = 0
        for i, a in enumerate(new):
            for p in range(lens[i], lens[i] + a):
                if p % page == 0:
                    n_free -= 1
                    table[i][p // page] = free[n_free]
                slots[t], positions[t] = table[i][p // page] * page + p % page, p
                t += 1
            lens[i] += a
            cu[i + 1] = t
    return table, lens, n_free, cu, slots, positions, status


def trim(table, lens, keep, free, n_free, page):
    status = 0
    back = []
    table, free = [list(r) for r in table], list(free)
    for i, (n, k) in enumerate(zip(lens, keep)):
        if n < 0 or k < 0:
            status |= 8
        elif k > n or n > len(table[0]) * page:
            status |= 2
        else:
            back += [(i, c) for c in range(pages_of(k, page), pages_of(n, page))]
    if n_free + len(back) > len(free):
        status |= 1
    if status == 0:
        for j, (i, c) in enumerate(back):
            free[n_free + len(back) - 1 - j] = table[i][c]
            table[i][c] = -1
        return table, list(keep), free, n_free + len(back), 0
    return table, list(lens), free, n_free, status


def rotate(x, positions, theta):
    """x [rows, heads, 128] in 64 bits."""
    half = D // 2
    freq = theta ** (-torch.arange(half, dtype=torch.float64) / half)
    angle = positions.double()[:, None] * freq
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def attention(q, k, v, table, lens, cu, hq, hkv):
    """(out, softmax @ |v|) in 64 bits; the second is what a rounding of the weights is measured against."""
    group, page = hq // hkv, k.shape[2]
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    out, mag = torch.zeros(q.shape[0], hq * D, dtype=torch.float64), torch.zeros(q.shape[0], hq * D, dtype=torch.float64)
    for i in range(len(lens)):
        new = cu[i + 1] - cu[i]
        if new <= 0 or lens[i] <= 0:
            continue
        pages = table[i][:pages_of(lens[i], page)]
        kk = k[pages].permute(1, 0, 2, 3).reshape(hkv, -1, D)[:, :lens[i]]
        vv = v[pages].permute(1, 0, 2, 3).reshape(hkv, -1, D)[:, :lens[i]]
        qq = q[cu[i]:cu[i + 1], :hq * D].reshape(new, hkv, group, D).permute(1, 0, 2, 3)
        s = torch.einsum("htgd,hpd->htgp", qq, kk) / math.sqrt(D)
        limit = lens[i] - new + torch.arange(new) + 1
        dark = (torch.arange(lens[i])[None] >= limit[:, None])[None, :, None]
        empty = (limit <= 0)[None, :, None, None]
        w = torch.softmax(s.masked_fill(dark, -math.inf), -1).masked_fill(empty, 0.0)
        for o, x in ((out, vv), (mag, vv.abs())):
            o[cu[i]:cu[i + 1]] = torch.einsum("htgp,hpd->htgd", w, x).permute(1, 0, 2, 3).reshape(new, hq * D)
    return out, mag


def verify(target, draft, tokens, lens, accept, sample):
    """Tensors on the CPU; draft None: certain drafts."""
    b, k = tokens.shape
    out, accepted = torch.full((b, k + 1), -1, dtype=torch.int64), torch.zeros(b, dtype=torch.int32)
    zero = lambda x: torch.where(x > 0, x, torch.zeros_like(x))  # NaN counts as nothing
    for r in range(b):
        n, most = 0, k if lens is None else max(0, min(k, int(lens[r])))
        while n < most:
            d = int(tokens[r, n])
            if not 0 <= d < target.shape[2]:
                break
            q = 1.0 if draft is None else float(draft[r, n, d])
            if not float(accept[r, n]) * q < float(target[r, n, d]):
                break
            n += 1
        p = target[r, n].double()
        w = zero(p)
        if n < most:
            if draft is None:
                left = w.clone()
                if 0 <= int(tokens[r, n]) < w.numel():
                    left[int(tokens[r, n])] = 0
            else:
                left = zero(p - draft[r, n].double())
            if left.sum() > 0:
                w = left
        cdf = w.cumsum(0)
        over = ((cdf > float(sample[r]) * cdf[-1]) & (w > 0)).nonzero()
        some = (w > 0).nonzero()
        out[r, :n] = tokens[r, :n]
        out[r, n] = over[0, 0] if len(over) else some[-1, 0] if len(some) else -1
        accepted[r] = n
    return out, accepted
