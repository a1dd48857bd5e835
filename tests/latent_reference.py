"""Latent attention from its definition in 64 bits, and how far a result may be off: shared by the tests."""
import math

import torch

ROPE, NOPE, VALUE = 64, 128, 128


def attend(q, keys, values, limits, scale):
    """q [n, d], keys [t, d], values [t, dv] (any type), limits: how many of the keys each row of q sees -> out [n, dv], lse [n], and for
    the tolerance sum p |v| [n, dv] and the largest sum |q k| scale of a row [n]; everything in 64 bits."""
    q, keys, values = q.double(), keys.double(), values.double()
    out = torch.zeros(q.shape[0], values.shape[1], dtype=torch.float64, device=q.device)
    mass, size, lse = out.clone(), torch.zeros_like(out[:, 0]), torch.full_like(out[:, 0], -math.inf)
    for limit in sorted(set(limits)):
        rows = [i for i, v in enumerate(limits) if v == limit]
        if limit <= 0:
            continue
        s = q[rows] @ keys[:limit].T * scale
        lse[rows] = torch.logsumexp(s, 1)
        p = torch.softmax(s, 1)
        out[rows], mass[rows] = p @ values[:limit], p @ values[:limit].abs()
        size[rows] = (q[rows].abs() @ keys[:limit].abs().T * abs(scale)).amax(1)
    return out, lse, mass, size


def check(got, got_lse, want, lse, mass, size, dtype, wide):
    """Half a rounding step of the output, half a step of every weight of the sum (the weights are rounded to the type for the second
    product, their sum is not), and the 32-bit errors: a score is the sum of ``wide`` products, added 16 at a time with an error of
    2^-23 of the sum so far at most, and moves its weight by as much, relatively, and the sum of the weights as well; exp2 and the running
    sums add less than 2^-18 for a hundred thousand positions; ``tiny`` is for weights and outputs below the type's normal numbers."""
    step = torch.finfo(dtype).eps / 2
    score = (wide / 16 + 4) * 2.0 ** -23 * size
    bound = step * want.abs() + (step + 2 * score[..., None] + 2.0 ** -18) * (mass + want.abs()) + torch.finfo(dtype).tiny
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"off by {float((err / bound).max()):.3g} of the bound"
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(got_lse) & (got_lse < 0), empty)
    bound = score + 2.0 ** -18 + 2.0 ** -23 * lse.abs()
    err = (got_lse.double() - lse).abs()
    assert bool((err <= bound)[~empty].all()), f"lse off by {float((err / bound)[~empty].max()):.3g} of the bound"
    assert not bool(got[empty].any())


def make_pool(lens, page, rank, dtype, gen, spare=3, layers=None, device="cuda", fill=None):
    """A pool with the pages of sequences of these lengths in no order -> cache, table (entries behind the last page: -7, never read), rows."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    cache = torch.randn(total, page, rank + ROPE, device=device, generator=gen).to(dtype)
    perm = torch.randperm(total, device=device, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32, device=device)
    at, rows = 0, []
    for i, (n, k) in enumerate(zip(lens, need)):
        table[i, :k] = perm[at:at + k]
        rows.append((table[i, :k].long(), n))
        at += k
    if fill is not None:  # rows that hold nothing: of the spare pages, and behind a sequence's end
        used = torch.zeros(total, page, dtype=torch.bool, device=device)
        for pages, n in rows:
            flat = torch.arange(len(pages) * page, device=device) < n
            used[pages] = flat.view(-1, page)
        cache[~used] = fill
    return cache, table, rows


def rows_of(cache, rows):
    pages, n = rows
    return cache[pages].flatten(0, 1)[:n]
