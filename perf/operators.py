"""Latent attention and its paged cache: the calls that are measured, over the range in which a server makes them.

One token of DeepSeek-V2's attention is cached as one row of ``rank + 64`` numbers that all heads share: the normalised
latent vector and the rotated part of the key.  ``latent_append`` makes and stores these rows, ``latent_decode`` attends
over them with the queries brought into the latent space (absorbed form), ``latent_decode_shared`` does so for groups of
sequences that begin with the same pages, ``latent_prefill`` attends over expanded keys and values of whole prompts, and
``copy_pages`` moves pages of all layers when sequences fork or the pool is compacted.

Where ``own`` is false the same results come from elementary tensor operations.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
ROPE, NOPE, VALUE = 64, 128, 128   # rotated part, unrotated key part and value of a head
SCALE = (NOPE + ROPE) ** -0.5
THETA, EPS = 1e4, 1e-6


def listed():
    return [
        # One sequence, one token, a few hundred positions: an interactive session's step, where latency counts.
        dict(name="decode_1", kind="decode", batch=1, steps=1, heads=16, rank=512, lo=700, hi=700, page=64, dtype="bf16"),
        # A server's batch of sequences of very different lengths.
        dict(name="decode_ragged", kind="decode", batch=37, steps=1, heads=16, rank=512, lo=60, hi=9000, page=64, dtype="bf16"),
        # Two sequences over whole documents, three drafted tokens each, small pages.
        dict(name="decode_long", kind="decode", batch=2, steps=3, heads=16, rank=512, lo=70001, hi=131072, page=32, dtype="fp16"),
        # A batch that shares a system prompt, each with a question of its own.
        dict(name="shared_prompt", kind="shared", batch=64, groups=1, steps=1, heads=16, rank=512, plo=8000, phi=8000, lo=1, hi=400,
             page=64, dtype="bf16"),
        # Several documents, each asked about by some of the batch; two drafted tokens each.
        dict(name="shared_groups", kind="shared", batch=21, groups=4, steps=2, heads=16, rank=512, plo=900, phi=5000, lo=2, hi=2500,
             page=64, dtype="fp16"),
        # A short prompt alone.
        dict(name="prefill_130", kind="prefill", heads=16, prompts="130", dtype="bf16"),
        # Prompts and pieces of prompts of a server's step, some behind positions that are there already.
        dict(name="prefill_ragged", kind="prefill", heads=16, prompts="1+4000 777 1500+513 64 350+1700 1404+2048",
             dtype="fp16"),
        # One long prompt.
        dict(name="prefill_8192", kind="prefill", heads=16, prompts="8192", dtype="bf16"),
        # The rows of a decode batch padded to a fixed size, far positions.
        dict(name="append_step", kind="append", tokens=40, padded=3, heads=16, rank=512, far=120000, page=64, dtype="bf16"),
        # The rows of a prompt.
        dict(name="append_prompt", kind="append", tokens=8191, padded=0, heads=16, rank=512, far=8191, page=64, dtype="fp16"),
        # A sequence forks: its last, partly filled page is copied in every layer.
        dict(name="pages_fork", kind="pages", layers=27, pool=64, copies=1, page=64, rank=512, dtype="bf16"),
        # A pool is compacted: many pages move down.
        dict(name="pages_compact", kind="pages", layers=27, pool=1200, copies=391, page=64, rank=512, dtype="bf16"),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng: random.Random):
    kind = rng.choice(("decode", "decode", "shared", "prefill", "prefill", "append", "pages"))
    dtype = rng.choice(("fp16", "bf16"))
    page = rng.choice((16, 32, 64, 64, 128))
    rank = rng.choice((256, 512, 512, 512))
    heads = rng.choice((5, 8, 16, 16, 16, 32, 128))
    if kind == "decode":
        batch, steps = _log_int(rng, 1, 128), rng.choice((1, 1, 2, 3, 5))
        hi = _log_int(rng, steps, max(steps, min(131072, 200000 // batch, 9000000 // (batch * steps * heads))))
        return dict(kind=kind, batch=batch, steps=steps, heads=heads, rank=rank, lo=max(steps, hi // rng.choice((1, 8, 100))), hi=hi, page=page,
                    dtype=dtype)
    if kind == "shared":
        batch, steps, heads = _log_int(rng, 2, 96), rng.choice((1, 1, 2, 4)), min(heads, 32)
        phi = _log_int(rng, 16, min(16384, 9000000 // (batch * steps * heads)))
        return dict(kind=kind, batch=batch, groups=rng.randint(1, min(batch, 4)), steps=steps, heads=heads, rank=rank, plo=max(1, phi // 2),
                    phi=phi, lo=4, hi=_log_int(rng, 4, 3000), page=page, dtype=dtype)
    if kind == "prefill":
        n = _log_int(rng, 1, 12)
        total = _log_int(rng, n, 7000)
        prompts = " ".join(f"{max(1, round(total / n * rng.uniform(0.1, 1.9)))}+{rng.choice((0, 0, _log_int(rng, 1, 3000)))}" for _ in range(n))
        return dict(kind=kind, heads=rng.choice((5, 8, 16)), prompts=prompts, dtype=dtype)
    if kind == "append":
        tokens = _log_int(rng, 1, 8192)
        return dict(kind=kind, tokens=tokens, padded=rng.randint(0, tokens // 4), heads=rng.choice((5, 8, 16, 32)), rank=rank,
                    far=_log_int(rng, tokens, 160000), page=page, dtype=dtype)
    layers = rng.choice((1, 5, 27))
    copies = _log_int(rng, 1, min(600, 650000 // (layers * page)))
    return dict(kind=kind, layers=layers, pool=2 * copies + rng.randint(1, 300), copies=copies, page=page, rank=rank,
                dtype=dtype)


# ---- what a user's program has in hand ------------------------------------------------------------
def _lengths(lo: int, hi: int, n: int):
    """Lengths spread over their logarithm from lo to hi, in an order that is not sorted."""
    v = [hi if n == 1 else round(lo * (hi / lo) ** (i / (n - 1))) for i in range(n)]
    random.Random(n).shuffle(v)
    return v


def _prompts(text: str):
    """"777 350+1700": new positions of each sequence, and those before them -> two lists."""
    parts = [[int(v) for v in p.split("+")] for p in text.split()]
    return [p[0] for p in parts], [p[1] if len(p) > 1 else 0 for p in parts]


def _starts(n: int, groups: int):
    return [round(i * n / groups) for i in range(groups + 1)]


def _generator(seed: int):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pool(case, lists, gen):
    """A pool of pages with some to spare, and the page tables of sequences of the given lengths: pages in no order,
    entries behind a sequence's last page zero."""
    page, width = case["page"], case["rank"] + ROPE
    need = [-(-n // page) for n in lists]
    pages = sum(need) + 3
    cache = torch.randn(pages, page, width, device="cuda", generator=gen).to(DTYPES[case["dtype"]])
    perm = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros(len(lists), max(max(need), 1), dtype=torch.int32, device="cuda")
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = perm[at:at + k]
        at += k
    return cache, table


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = _generator(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dt)

    s = SimpleNamespace(kind=kind)
    if kind in ("decode", "shared"):
        B, S, H, R = case["batch"], case["steps"], case["heads"], case["rank"]
        lens = _lengths(case["lo"], case["hi"], B)
        prefix = _lengths(case["plo"], case["phi"], case["groups"]) if kind == "shared" else []
        s.cache, table = _pool(case, lens + prefix, gen)
        s.table, s.lens = table[:B].contiguous(), _ints(lens)
        # what the absorbing product leaves: one [rows, rank] block a head, seen as [batch, steps, heads, rank]
        s.q_latent = randn(H, B * S, R).view(H, B, S, R).permute(1, 2, 0, 3)
        s.q_rope = randn(B, S, H, ROPE)
        if kind == "shared":
            s.prefix_table, s.prefix_lens = table[B:].contiguous(), _ints(prefix)
            s.starts = _ints(_starts(B, case["groups"]))
    elif kind == "prefill":
        H, (new, old) = case["heads"], _prompts(case["prompts"])
        total = [a + b for a, b in zip(new, old)]
        s.q = randn(sum(new), H, NOPE + ROPE)
        s.q_rope = randn(sum(new), H, ROPE)
        s.kv = randn(sum(total), H, NOPE + VALUE)
        s.k_rope = randn(sum(total), ROPE)
        s.most_new, s.most_keys = max(new), max(total)
        s.cu_q = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        s.cu_k = _ints([sum(total[:i]) for i in range(len(new) + 1)])
    elif kind == "append":
        T, H, R = case["tokens"], case["heads"], case["rank"]
        pages = -(-T // case["page"]) + 2
        s.cache = randn(pages, case["page"], R + ROPE)
        s.kv = 3 * randn(T, R + ROPE)
        s.q = randn(T, H, NOPE + ROPE)
        s.weight = (1 + 0.1 * torch.randn(R, device="cuda", generator=gen)).to(dt)
        s.inv_freq = 1.0 / THETA ** (torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float32) / ROPE)
        s.positions = torch.randint(0, case["far"], (T,), device="cuda", generator=gen)
        s.slots = torch.randperm(pages * case["page"], device="cuda", generator=gen)[:T]
        if case["padded"]:
            s.slots[-case["padded"]:] = -1
    else:
        s.cache = randn(case["layers"], case["pool"], case["page"], case["rank"] + ROPE)
        perm = torch.randperm(case["pool"], device="cuda", generator=gen)
        s.src, s.dst = perm[:case["copies"]].clone(), perm[case["copies"]:2 * case["copies"]].clone()
    return s


# ---- one pass ---------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from gemq_b200 import kernels as K
    if s.kind == "decode":
        return K.latent_decode(s.q_latent, s.q_rope, s.cache, s.table, s.lens, SCALE)
    if s.kind == "shared":
        return K.latent_decode_shared(s.q_latent, s.q_rope, s.cache, s.table, s.lens, s.prefix_table, s.prefix_lens, s.starts, SCALE)
    if s.kind == "prefill":
        return K.latent_prefill(s.q[..., :NOPE], s.q_rope, s.kv, s.k_rope, s.cu_q, s.cu_k, SCALE)
    if s.kind == "append":
        q_rope, rows = K.latent_append(s.kv, s.q[..., NOPE:], s.weight, EPS, s.inv_freq, s.positions, s.slots, s.cache)
        return q_rope, rows, s.cache
    K.copy_pages(s.cache, s.src, s.dst)
    return s.cache


def _softmax_sum(scores, hidden, values):
    """scores and hidden [.., rows, keys], values [.., keys, dv] -> out and the logarithm of the sum; rows that see nothing: 0, -inf."""
    scores = scores.masked_fill(hidden, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    empty = top == float("-inf")
    p = torch.exp(scores - top.masked_fill(empty, 0.0))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / total.masked_fill(empty, 1.0)
    return out, (top + torch.log(total.masked_fill(empty, 1.0))).squeeze(-1)


def _rotate(x, positions, inv_freq):
    """Neighbouring numbers are a pair; the angle is formed in 64 bits: far positions times a frequency lose it in 32."""
    angle = positions.double()[:, None] * inv_freq.double()[None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    if x.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _plain_decode(s):
    """The batch padded to its longest sequence: a shared prefix is one more block of keys in front of each sequence's own."""
    B, S, H, R = s.q_latent.shape
    page = s.cache.shape[1]
    device = s.cache.device
    keys = s.cache[s.table.long()].flatten(1, 2)
    at = torch.arange(keys.shape[1], device=device).expand(B, -1)
    length, there = s.lens.long()[:, None], at < s.lens[:, None]
    if s.kind == "shared":
        group = torch.searchsorted(s.starts, torch.arange(B, device=device, dtype=torch.int32), right=True) - 1
        before = s.prefix_lens.long()[group][:, None]
        keys = torch.cat([s.cache[s.prefix_table.long()[group]].flatten(1, 2), keys], 1)
        first = torch.arange(s.prefix_table.shape[1] * page, device=device).expand(B, -1)
        at, there = torch.cat([first, at + before], 1), torch.cat([first < before, there], 1)
        length = length + before
    limits = length - (S - 1) + torch.arange(S, device=device)
    hidden = ~there[:, None, :] | (at[:, None, :] >= limits[:, :, None])  # [B, S, keys]
    keys = keys.float()
    q = torch.cat([s.q_latent, s.q_rope], -1).float().flatten(1, 2)
    scores = torch.matmul(q, keys.transpose(1, 2)) * SCALE
    out, lse = _softmax_sum(scores, hidden.repeat_interleave(H, 1), keys[..., :R])
    return out.view(B, S, H, R).to(s.q_latent.dtype), lse.view(B, S, H)


def _plain_prefill(s):
    """The prompts padded to the longest."""
    device = s.q.device
    cu_q, cu_k = s.cu_q.long(), s.cu_k.long()
    new, total = cu_q.diff()[:, None], cu_k.diff()[:, None]
    i, j = torch.arange(s.most_new, device=device), torch.arange(s.most_keys, device=device)
    rows = (cu_q[:-1, None] + i).clamp(max=s.q.shape[0] - 1)
    keys = (cu_k[:-1, None] + j).clamp(max=s.kv.shape[0] - 1)
    q = torch.cat([s.q[..., :NOPE], s.q_rope], -1)[rows].float().transpose(1, 2)
    kv = s.kv[keys].float().transpose(1, 2)
    rope = s.k_rope[keys].float()[:, None].expand(-1, kv.shape[1], -1, -1)
    scores = torch.matmul(q, torch.cat([kv[..., :NOPE], rope], -1).transpose(-1, -2)) * SCALE
    hidden = (j[None, None, :] >= (total - new + 1 + i)[:, :, None]) | (j >= total)[:, None, :]
    out, lse = _softmax_sum(scores, hidden[:, None], kv[..., NOPE:])
    row = torch.arange(s.q.shape[0], device=device)
    seq = torch.searchsorted(cu_q, row, right=True) - 1
    row = row - cu_q[seq]
    return out[seq, :, row].to(s.q.dtype), lse[seq, :, row]


def _run_plain(s):
    if s.kind in ("decode", "shared"):
        return _plain_decode(s)
    if s.kind == "prefill":
        return _plain_prefill(s)
    if s.kind == "append":
        R = s.weight.shape[0]
        c = s.kv[:, :R].float()
        c = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * s.weight.float()
        rows = torch.cat([c, _rotate(s.kv[:, R:].float(), s.positions, s.inv_freq)], -1).to(s.kv.dtype)
        keep = s.slots >= 0
        s.cache.view(-1, rows.shape[1])[s.slots[keep]] = rows[keep]
        return _rotate(s.q[..., NOPE:].float(), s.positions, s.inv_freq).to(s.q.dtype), rows, s.cache
    s.cache[:, s.dst] = s.cache[:, s.src]
    return s.cache


# ---- the definition in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "pages":
        want = s.cache.clone()
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            want[:, b].copy_(s.cache[:, a])
        return want
    if kind == "append":
        R = case["rank"]
        x = s.kv.double()
        norm = torch.sqrt(x[:, :R].pow(2).sum(1) / R + EPS)
        latent = x[:, :R] / norm[:, None] * s.weight.double()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s.positions.double()[:, None] * s.inv_freq.double())
        def rot(v, t):
            return torch.view_as_real(torch.view_as_complex(v.unflatten(-1, (-1, 2)).contiguous()) * t).flatten(-2)
        rows = torch.cat([latent, rot(x[:, R:], turn)], 1)
        cache = s.cache.double()
        flat = cache.view(-1, R + ROPE)
        for t, slot in enumerate(s.slots.tolist()):
            if slot >= 0:
                flat[slot] = rows[t]
        return rot(s.q[..., NOPE:].double(), turn[:, None]), rows, cache

    def softmax_sum(scores, values):
        """Weights by the sum of exponentials of each row -> out, log of the sum; rows that see nothing: 0, -inf."""
        lse = torch.logsumexp(scores, -1)
        w = torch.exp(scores - torch.where(lse.isinf(), torch.zeros_like(lse), lse)[..., None])
        return w @ values, lse

    if kind == "prefill":
        out = torch.zeros(*s.q.shape[:2], VALUE, dtype=torch.float64, device="cuda")
        lse = torch.zeros(s.q.shape[:2], dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for new, old in zip(*_prompts(case["prompts"])):
            seen = torch.ones(new, new + old, dtype=torch.bool, device="cuda").tril(old)
            for h in range(case["heads"]):
                kv = s.kv[k0:k0 + new + old, h].double()
                scores = s.q[q0:q0 + new, h, :NOPE].double() @ kv[:, :NOPE].T
                scores += s.q_rope[q0:q0 + new, h].double() @ s.k_rope[k0:k0 + new + old].double().T
                scores = torch.where(seen, scores * SCALE, -math.inf)
                out[q0:q0 + new, h], lse[q0:q0 + new, h] = softmax_sum(scores, kv[:, NOPE:])
            q0, k0 = q0 + new, k0 + new + old
        return out, lse

    B, S, H, R, page = case["batch"], case["steps"], case["heads"], case["rank"], case["page"]
    lens = _lengths(case["lo"], case["hi"], B)
    out = torch.zeros(B, S, H, R, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, S, H, dtype=torch.float64, device="cuda")
    group = [0] * B
    if kind == "shared":
        prefix, starts = _lengths(case["plo"], case["phi"], case["groups"]), _starts(B, case["groups"])
        for g in range(case["groups"]):
            group[starts[g]:starts[g + 1]] = [g] * (starts[g + 1] - starts[g])
    for b in range(B):
        lists = [(s.table[b], lens[b])]
        if kind == "shared":
            lists.insert(0, (s.prefix_table[group[b]], prefix[group[b]]))
        tokens = torch.cat([s.cache[t.long()].reshape(-1, R + ROPE)[:n] for t, n in lists]).double()
        for i in range(S):
            seen = tokens[:max(len(tokens) - (S - 1 - i), 0)]
            scores = SCALE * (s.q_latent[b, i].double() @ seen[:, :R].T + s.q_rope[b, i].double() @ seen[:, R:].T)
            if len(seen):
                out[b, i], lse[b, i] = softmax_sum(scores, seen[:, :R])
            else:
                lse[b, i] = -math.inf
    return out, lse


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("decode", "shared"):
        rows, width = case["steps"] * case["heads"], case["rank"] + ROPE
        lens = _lengths(case["lo"], case["hi"], case["batch"])
        tokens, pairs = sum(lens), rows * sum(lens)
        if kind == "shared":
            prefix, starts = _lengths(case["plo"], case["phi"], case["groups"]), _starts(case["batch"], case["groups"])
            tokens += sum(prefix)
            pairs += rows * sum(n * (b - a) for n, a, b in zip(prefix, starts, starts[1:]))
        rows *= case["batch"]
        return dict(bytes=2 * (tokens * width + rows * (width + case["rank"])) + 4 * rows, flops=2 * pairs * (width + case["rank"]))
    if kind == "prefill":
        H, (new, old) = case["heads"], _prompts(case["prompts"])
        seen = sum(n * o + n * (n + 1) // 2 for n, o in zip(new, old))
        keys = sum(new) + sum(old)
        return dict(bytes=2 * (sum(new) * H * (NOPE + ROPE + VALUE) + keys * (H * (NOPE + VALUE) + ROPE)) + 4 * sum(new) * H,
                    flops=2 * seen * H * (NOPE + ROPE + VALUE))
    if kind == "append":
        T, width = case["tokens"], case["rank"] + ROPE
        return dict(bytes=2 * ((3 * T - case["padded"]) * width + 2 * T * case["heads"] * ROPE) + 16 * T,
                    flops=T * (5 * case["rank"] + 3 * ROPE * (1 + case["heads"])))
    page = case["page"] * (case["rank"] + ROPE) * 2
    return dict(bytes=2 * case["layers"] * case["copies"] * page, flops=0)
