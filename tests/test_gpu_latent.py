"""Latent attention, its cache and page copies against their definitions in 64 bits."""
import math

import pytest
import torch

from latent_reference import NOPE, ROPE, VALUE, attend, check, make_pool, rows_of

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def nothing_reported():
    from gemq_b200.kernels import latent_error
    latent_error()
    yield
    assert latent_error() == 0


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- decoded tokens ---------------------------------------------------------------------------------
def decode_case(lens, S, H, R, page, dtype, seed=0, fill=NAN, spread=1.0):
    gen = generator(seed)
    cache, table, rows = make_pool(lens, page, R, dtype, gen, fill=fill)
    B = len(lens)
    q_latent = (spread * torch.randn(H, B * S, R, device="cuda", generator=gen)).to(dtype).view(H, B, S, R).permute(1, 2, 0, 3)
    q_rope = (spread * torch.randn(B, S, H, ROPE, device="cuda", generator=gen)).to(dtype)
    return q_latent, q_rope, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), rows


def check_decode(got, lse, q_latent, q_rope, tokens, scale):
    B, S, H, R = q_latent.shape
    assert got.shape == q_latent.shape and got.dtype == q_latent.dtype and lse.shape == (B, S, H) and lse.dtype == torch.float32
    q = torch.cat([q_latent, q_rope], -1)
    for b in range(B):
        limits = [len(tokens[b]) - (S - 1 - i) for i in range(S) for _ in range(H)]
        want = attend(q[b].flatten(0, 1), tokens[b], tokens[b][:, :R], limits, scale)
        check(got[b].flatten(0, 1), lse[b].flatten(), *want, got.dtype, R + ROPE)


DECODE = [
    # lens, steps, heads, rank, page
    ([1], 1, 16, 512, 64),
    ([0, 5, 64, 65, 0, 128, 63], 1, 16, 512, 64),           # empty sequences, whole pages, one row on a page
    ([700], 1, 16, 512, 16),
    ([1000, 17, 48, 49], 1, 5, 512, 16),                    # an odd number of heads; pages that end inside a tile
    ([300, 31, 32, 33], 2, 16, 256, 32),
    ([2, 1, 0, 3, 200], 3, 8, 512, 64),                     # more steps than positions: rows that see nothing
    ([257, 900], 5, 16, 128, 128),                          # 80 rows a sequence
    ([400, 129], 1, 128, 512, 64),
    ([511, 64], 2, 33, 384, 192),
    ([5000, 40, 3000], 1, 16, 512, 64),
    ([20000], 1, 1, 512, 64),
    ([130] * 70, 1, 16, 512, 64),
    ([1 + 37 * i % 400 for i in range(200)], 1, 4, 128, 16),
    ([i % 3 * 50 for i in range(1000)], 1, 3, 128, 64),      # more sequences than threads
    ([130, 45], 40, 16, 256, 32),                            # a piece of a prompt: 640 rows a sequence, some that see nothing
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,S,H,R,page", DECODE)
def test_decode(lens, S, H, R, page, dtype):
    """Rows of the pool that hold nothing are NaN: they must not be seen."""
    from gemq_b200.kernels import latent_decode
    q_latent, q_rope, cache, table, n, rows = decode_case(lens, S, H, R, page, dtype, seed=len(lens) + S)
    scale = 192 ** -0.5
    before = cache.clone()
    got, lse = latent_decode(q_latent, q_rope, cache, table, n, scale)
    check_decode(got, lse, q_latent, q_rope, [rows_of(cache, r) for r in rows], scale)
    assert torch.equal(before.view(torch.int16), cache.view(torch.int16))
    again, lse2 = latent_decode(q_latent, q_rope, cache, table, n, scale)
    assert torch.equal(got, again) and torch.equal(lse, lse2)  # the order of the sums does not change


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_of_steep_scores(dtype):
    """Scores of hundreds that grow along the sequence (the running maximum moves again and again), and their opposite."""
    from gemq_b200.kernels import latent_decode
    for sign in (1, -1):
        q_latent, q_rope, cache, table, n, rows = decode_case([1500, 90], 2, 16, 512, 64, dtype, seed=3, fill=0.0, spread=3.0)
        ramp = torch.linspace(0.1, 2.0, 1500, device="cuda")
        pages, length = rows[0]
        flat = cache[pages].flatten(0, 1)
        base = q_latent[0, 0, 0]
        flat[:length, :512] = (sign * ramp[:, None] * base.float()[None] * 0.3 + 0.1 * flat[:length, :512].float()).to(dtype)
        cache[pages] = flat.view(len(pages), 64, -1)
        got, lse = latent_decode(q_latent, q_rope, cache, table, n, 192 ** -0.5)
        check_decode(got, lse, q_latent, q_rope, [rows_of(cache, r) for r in rows], 192 ** -0.5)


@pytest.mark.parametrize("value", [NAN, INF, -INF, 65504.0])
@pytest.mark.parametrize("S,n", [(1, 100), (4, 100), (4, 66), (3, 2), (9, 128)])
def test_decode_sees_nothing_behind_its_position(S, n, value):
    """Rows behind what a query sees have no influence on it, those of the later queries among them; a query that sees a NaN is NaN."""
    from gemq_b200.kernels import latent_decode
    q_latent, q_rope, cache, table, lens, rows = decode_case([n, 70], S, 16, 512, 64, torch.float16, seed=S)
    scale = 192 ** -0.5
    want, want_lse = latent_decode(q_latent, q_rope, cache, table, lens, scale)
    bad = cache.clone()
    pages, _ = rows[0]
    hit = max(n - (S - 1) // 2 - 1, 0)  # the last rows of the draft, from the one in its middle
    flat = bad[pages].flatten(0, 1)
    flat[hit:] = value
    bad[pages] = flat.view(len(pages), 64, -1)
    got, lse = latent_decode(q_latent, q_rope, bad, table, lens, scale)
    blind = [i for i in range(S) if n - (S - 1 - i) <= hit]
    seeing = [i for i in range(S) if n - (S - 1 - i) > hit]
    assert torch.equal(got[1], want[1]) and torch.equal(lse[1], want_lse[1])
    assert torch.equal(got[0, blind], want[0, blind]) and torch.equal(lse[0, blind], want_lse[0, blind])
    if math.isnan(value):
        assert bool(got[0, seeing].isnan().all())


def test_decode_without_a_row():
    """No sequence has one, in a table with and without room."""
    from gemq_b200.kernels import latent_decode
    for width in (0, 3):
        cache = torch.full((4, 64, 576), NAN, dtype=torch.float16, device="cuda")
        table = torch.full((2, width), 99, dtype=torch.int32, device="cuda")
        q = torch.ones(2, 2, 16, 512, dtype=torch.float16, device="cuda")
        out, lse = latent_decode(q, q[..., :64], cache, table, torch.zeros(2, dtype=torch.int32, device="cuda"), 0.1)
        assert not bool(out.any()) and bool((lse == -INF).all())
    out, lse = latent_decode(q[:0], q[:0, ..., :64], cache, table[:0], torch.zeros(0, dtype=torch.int32, device="cuda"), 0.1)
    assert out.shape == (0, 2, 16, 512) and lse.shape == (0, 2, 16)


@pytest.mark.parametrize("value", [NAN, INF])
def test_a_querys_nan_is_its_own(value):
    from gemq_b200.kernels import latent_decode, latent_prefill
    q_latent, q_rope, cache, table, lens, _ = decode_case([700, 90], 2, 16, 512, 64, torch.bfloat16)
    want = latent_decode(q_latent, q_rope, cache, table, lens, 0.07)
    bad = q_latent.clone()
    bad[0, 1, 5, 3] = value
    got = latent_decode(bad, q_rope, cache, table, lens, 0.07)
    keep = torch.ones(2, 2, 16, dtype=torch.bool, device="cuda")
    keep[0, 1, 5] = False
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, want)) and bool(got[0][0, 1, 5].isnan().all())
    q, kv, k_rope, cu_q, cu_k = prefill_case([(300, 400)], 2, torch.bfloat16)
    want = latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, 0.07)
    bad = q.clone()
    bad[140, 1, 7] = value
    got = latent_prefill(bad[..., :NOPE], bad[..., NOPE:], kv, k_rope, cu_q, cu_k, 0.07)
    keep = torch.ones(300, 2, dtype=torch.bool, device="cuda")
    keep[140, 1] = False
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, want)) and bool(got[0][140, 1].isnan().all())


@pytest.mark.parametrize("scale", [-0.05, 0.0, 3.0])
def test_scales(scale):
    from gemq_b200.kernels import latent_decode, latent_prefill
    q_latent, q_rope, cache, table, lens, rows = decode_case([200, 65], 1, 16, 512, 64, torch.float16)
    got, lse = latent_decode(q_latent, q_rope, cache, table, lens, scale)
    check_decode(got, lse, q_latent, q_rope, [rows_of(cache, r) for r in rows], scale)
    q, kv, k_rope, cu_q, cu_k = prefill_case([(150, 150)], 2, torch.float16)
    got, lse = latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, scale)
    check_prefill(got, lse, [(150, 150)], q, kv, k_rope, scale, True)


def test_prefill_without_a_key():
    from gemq_b200.kernels import latent_prefill
    q, kv, k_rope, cu_q, cu_k = prefill_case([(150, 0), (3, 0)], 2, torch.float16)
    for causal in (True, False):
        out, lse = latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, 0.1, causal)
        assert not bool(out.any()) and bool((lse == -INF).all())
    q, kv, k_rope, cu_q, cu_k = prefill_case([(0, 5)], 2, torch.float16)
    assert latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, 0.1)[0].shape == (0, 2, 128)
    q, kv, k_rope, cu_q, cu_k = prefill_case([], 2, torch.float16, spare=4)  # rows, but no sequences
    out, lse = latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, 0.1)
    assert not bool(out.any()) and bool((lse == -INF).all())


def test_prefill_of_expanded_tensors():
    """One query head and one key head seen as several (strides of 0)."""
    from gemq_b200.kernels import latent_prefill
    q, kv, k_rope, cu_q, cu_k = prefill_case([(90, 130)], 1, torch.float16)
    want = latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, 0.07)
    got = latent_prefill(q[..., :NOPE].expand(-1, 3, -1), q[..., NOPE:].expand(-1, 3, -1), kv.expand(-1, 3, -1), k_rope, cu_q, cu_k, 0.07)
    assert all(torch.equal(a.expand(b.shape) if a.dim() == 3 else a.expand(-1, 3), b) for a, b in zip(want, got))


def test_decode_takes_any_strides():
    from gemq_b200.kernels import latent_decode
    q_latent, q_rope, cache, table, lens, _ = decode_case([100, 333], 2, 8, 512, 64, torch.bfloat16)
    want = latent_decode(q_latent, q_rope, cache, table, lens, 0.07)
    layers = torch.full((cache.shape[0], 3, 64, 576), NAN, dtype=cache.dtype, device="cuda")
    layers[:, 1] = cache
    joined = torch.cat([q_latent, q_rope], -1)
    got = latent_decode(joined[..., :512], joined[..., 512:], layers[:, 1], table, lens, 0.07)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = latent_decode(q_latent[:1], q_rope[:1], cache, table[:1], lens[:1], 0.07)
    check_decode(*one, q_latent[:1], q_rope[:1], [rows_of(cache, (table[0, :2].long(), 100))], 0.07)
    got = latent_decode(q_latent[:, :1].expand(-1, 2, -1, -1), q_rope[:, :1].expand(-1, 2, -1, -1), cache, table, lens, 0.07)
    assert torch.equal(got[0][:, 0], want[0][:, 0])


def test_decode_far_pages():
    """A pool beyond 2^31 elements: rows at its end, and the same ones near its beginning."""
    from gemq_b200.kernels import latent_decode
    pages = 2 ** 31 // (64 * 576) + 40
    pool = torch.empty(pages, 64, 576, dtype=torch.float16, device="cuda")
    gen = generator(1)
    data = torch.randn(8, 64, 576, device="cuda", generator=gen).half()
    pool[:8], pool[-8:] = data, data
    q_latent = torch.randn(2, 1, 16, 512, device="cuda", generator=gen).half()
    q_latent[1] = q_latent[0]
    q_rope = torch.randn(1, 1, 16, 64, device="cuda", generator=gen).half().expand(2, -1, -1, -1)
    near = torch.arange(8, device="cuda", dtype=torch.int32)
    table = torch.stack([near, near + (pages - 8)])
    lens = torch.tensor([500, 500], dtype=torch.int32, device="cuda")
    out, lse = latent_decode(q_latent, q_rope, pool, table, lens, 0.07)
    assert torch.equal(out[0], out[1]) and torch.equal(lse[0], lse[1])
    check_decode(out[1:], lse[1:], q_latent[1:], q_rope[1:], [data.flatten(0, 1)[:500]], 0.07)


def test_decode_reports_bad_pages_and_lengths():
    from gemq_b200.kernels import latent_decode, latent_error
    q_latent, q_rope, cache, table, lens, _ = decode_case([100, 300, 64], 1, 16, 512, 64, torch.bfloat16, fill=0.0)
    want, want_lse = latent_decode(q_latent, q_rope, cache, table, lens, 0.07)
    for bad in (cache.shape[0], -1, 2 ** 31 - 1):
        t = table.clone()
        t[1, 2] = bad
        got, lse = latent_decode(q_latent, q_rope, cache, t, lens, 0.07)
        assert latent_error() == 41
        assert bool(got[1].isnan().all()) and bool(lse[1].isnan().all())
        assert torch.equal(got[[0, 2]], want[[0, 2]]) and torch.equal(lse[[0, 2]], want_lse[[0, 2]])
    n = lens.clone()
    n[2] = -5
    got, lse = latent_decode(q_latent, q_rope, cache, table, n, 0.07)
    assert latent_error() == 42
    assert not bool(got[2].any()) and bool((lse[2] == -INF).all()) and torch.equal(got[:2], want[:2])
    n = lens.clone()
    n[1] = 10 ** 9  # as long as its table
    got, lse = latent_decode(q_latent, q_rope, cache, table, n, 0.07)
    assert latent_error() == 42
    n[1] = table.shape[1] * 64
    want, _ = latent_decode(q_latent, q_rope, cache, table, n, 0.07)
    assert torch.equal(got, want)


# ---- groups with a prefix -----------------------------------------------------------------------------
SHARED = [
    # prefix lengths, sequences of each group, own lengths (cycled), steps, heads, rank, page
    ([500], [3], [1, 64, 100], 1, 16, 512, 64),
    ([64, 0, 130], [2, 1, 3], [5, 70, 0, 33], 1, 16, 512, 64),    # a group without a prefix, a sequence without rows of its own
    ([1000, 33], [9, 4], [1, 2, 40], 4, 8, 256, 16),              # fewer own rows than steps: the prefix's end is hidden
    ([2, 1], [2, 2], [0, 1], 3, 5, 512, 32),
    ([3000], [70], [1 + 13 * i % 90 for i in range(70)], 1, 16, 512, 64),
    ([700, 300, 50], [0, 5, 0], [20], 2, 16, 128, 64),            # groups without sequences
    ([400], [1], [300], 1, 128, 512, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix,sizes,own,S,H,R,page", SHARED)
def test_decode_shared(prefix, sizes, own, S, H, R, page, dtype):
    from gemq_b200.kernels import latent_decode_shared
    B, G = sum(sizes), len(sizes)
    lens = [own[b % len(own)] for b in range(B)]
    q_latent, q_rope, cache, table, n, rows = decode_case(lens + prefix, S, H, R, page, dtype, seed=B)
    q_latent, q_rope = q_latent[:B], q_rope[:B]
    starts = [sum(sizes[:g]) for g in range(G + 1)]
    scale = 192 ** -0.5
    args = (q_latent, q_rope, cache, table[:B].contiguous(), n[:B].contiguous(), table[B:].contiguous(), n[B:].contiguous(),
            torch.tensor(starts, dtype=torch.int32, device="cuda"), scale)
    got, lse = latent_decode_shared(*args)
    tokens = []
    for b in range(B):
        g = max(g for g in range(G) if starts[g] <= b and sizes[g])
        tokens.append(torch.cat([rows_of(cache, rows[B + g]), rows_of(cache, rows[b])]))
    check_decode(got, lse, q_latent, q_rope, tokens, scale)
    again, lse2 = latent_decode_shared(*args)
    assert torch.equal(got, again) and torch.equal(lse, lse2)


def test_decode_shared_sees_nothing_behind_its_position():
    """A draft longer than a sequence's own rows: what the earlier queries do not see of the prefix does not touch them."""
    from gemq_b200.kernels import latent_decode_shared
    q_latent, q_rope, cache, table, n, rows = decode_case([1, 30, 100], 4, 16, 512, 64, torch.bfloat16, seed=2)
    args = lambda c: (q_latent[:2], q_rope[:2], c, table[:2], n[:2], table[2:].contiguous(), n[2:].contiguous(),  # noqa: E731
                      torch.tensor([0, 2], dtype=torch.int32, device="cuda"), 0.07)
    want, _ = latent_decode_shared(*args(cache))
    bad = cache.clone()
    pages, _ = rows[2]
    bad[pages[99 // 64], 99 % 64] = NAN  # the prefix's last row: seen by the first sequence's queries 2 and 3 and all of the second's
    got, _ = latent_decode_shared(*args(bad))
    assert torch.equal(got[0, :2], want[0, :2])
    assert bool(got[0, 2:].isnan().all()) and bool(got[1].isnan().all())


def test_decode_shared_reports_bad_tables():
    from gemq_b200.kernels import latent_decode_shared, latent_error
    q_latent, q_rope, cache, table, n, rows = decode_case([10, 20, 30, 300, 200], 1, 16, 512, 64, torch.bfloat16, fill=0.0)
    base = dict(q_latent=q_latent[:3], q_rope=q_rope[:3], cache=cache, table=table[:3].contiguous(), lens=n[:3].contiguous(),
                prefix_table=table[3:].contiguous(), prefix_lens=n[3:].contiguous(),
                starts=torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda"), scale=0.07)
    want, _ = latent_decode_shared(**base)
    t = base["prefix_table"].clone()
    t[0, 1] = 10 ** 8
    got, _ = latent_decode_shared(**{**base, "prefix_table": t})
    assert latent_error() == 41 and bool(got[:2].isnan().all()) and torch.equal(got[2], want[2])
    for starts in ([0, 2, 99], [-4, 2, 3], [0, 50, 3], [0, -1, 3], [1, 2, 3], [0, 2, 2]):  # nothing is read or written out of range
        latent_decode_shared(**{**base, "starts": torch.tensor(starts, dtype=torch.int32, device="cuda")})
        assert latent_error() == 42, starts


# ---- prompts ------------------------------------------------------------------------------------------
PREFILL = [
    # (queries, keys) of the sequences, heads
    ([(1, 1)], 16),
    ([(1, 700), (130, 130)], 16),
    ([(127, 127), (128, 128), (129, 129), (1, 1), (0, 0), (64, 300)], 4),
    ([(5, 3), (4, 0), (0, 10), (300, 100)], 3),       # queries that see nothing; keys without queries
    ([(700, 1000)], 5),
    ([(256, 256), (257, 512), (255, 1023)], 2),
    ([(1500, 1500)], 2),
    ([(3, 5)] * 90, 2),
    ([(i % 7 * 50, i % 5 * 90) for i in range(150)], 1),   # several times 32 sequences, some without queries, some without keys
]


def prefill_case(parts, H, dtype, seed=0, spare=0):
    gen = generator(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    Tq, Tk = sum(p[0] for p in parts), sum(p[1] for p in parts)
    q = randn(Tq + spare, H, NOPE + ROPE)
    kv, k_rope = randn(Tk, H, NOPE + VALUE), randn(Tk, ROPE)
    cu = [torch.tensor([sum(p[k] for p in parts[:i]) for i in range(len(parts) + 1)], dtype=torch.int32, device="cuda") for k in (0, 1)]
    return q, kv, k_rope, cu[0], cu[1]


def check_prefill(got, lse, parts, q, kv, k_rope, scale, causal):
    H = q.shape[1]
    assert got.shape == (q.shape[0], H, VALUE) and got.dtype == q.dtype and lse.dtype == torch.float32 and lse.shape == got.shape[:2]
    q0 = k0 = 0
    for n, t in parts:
        limits = [t - n + 1 + i if causal else t for i in range(n)]
        for h in range(H):
            keys = torch.cat([kv[k0:k0 + t, h, :NOPE], k_rope[k0:k0 + t]], -1)
            if causal and n > 40 and t:  # row by row takes long: the same in one masked product
                want = masked(q[q0:q0 + n, h], keys, kv[k0:k0 + t, h, NOPE:], limits, scale)
            else:
                want = attend(q[q0:q0 + n, h], keys, kv[k0:k0 + t, h, NOPE:], limits, scale)
            check(got[q0:q0 + n, h], lse[q0:q0 + n, h], *want, got.dtype, NOPE + ROPE)
        q0, k0 = q0 + n, k0 + t


def masked(q, keys, values, limits, scale):
    q, keys, values = q.double(), keys.double(), values.double()
    limits = torch.tensor(limits, device=q.device)
    hidden = torch.arange(keys.shape[0], device=q.device)[None] >= limits[:, None]
    s = (q @ keys.T * scale).masked_fill(hidden, -INF)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse.clamp(min=-1e300)[:, None]).masked_fill(hidden, 0.0)
    size = (q.abs() @ keys.abs().T * abs(scale)).masked_fill(hidden, 0.0).amax(1)
    return p @ values, lse, p @ values.abs(), size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("parts,H", PREFILL)
def test_prefill(parts, H, causal, dtype):
    from gemq_b200.kernels import latent_prefill
    q, kv, k_rope, cu_q, cu_k = prefill_case(parts, H, dtype, seed=H, spare=3)
    scale = 192 ** -0.5
    got, lse = latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, scale, causal)
    check_prefill(got, lse, parts, q, kv, k_rope, scale, causal)
    assert not bool(got[-3:].any()) and bool((lse[-3:] == -INF).all())  # rows behind the last sequence
    again, lse2 = latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, scale, causal)
    assert torch.equal(got, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefill_of_steep_scores(dtype):
    from gemq_b200.kernels import latent_prefill
    parts = [(400, 900)]
    q, kv, k_rope, cu_q, cu_k = prefill_case(parts, 2, dtype)
    for sign in (1, -1):
        ramp = torch.linspace(0.1, 6.0, 900, device="cuda") * sign
        kv[:, 0, :NOPE] = (ramp[:, None] * q[7, 0, :NOPE].float() + 0.1 * kv[:, 0, :NOPE].float()).to(dtype)
        got, lse = latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, 192 ** -0.5)
        check_prefill(got, lse, parts, q, kv, k_rope, 192 ** -0.5, True)


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("at", [0, 63, 64, 127, 128, 200, 299])
def test_prefill_sees_nothing_behind_its_position(at, value):
    """A row's keys and values have no influence on the queries before it, nor on other sequences."""
    from gemq_b200.kernels import latent_prefill
    parts = [(300, 300), (77, 77), (260, 300)]
    q, kv, k_rope, cu_q, cu_k = prefill_case(parts, 2, torch.bfloat16)
    args = lambda kv, kr: (q[..., :NOPE], q[..., NOPE:], kv, kr, cu_q, cu_k, 0.07)  # noqa: E731
    want, want_lse = latent_prefill(*args(kv, k_rope))
    for where in ("keys", "values", "rope"):
        bad, rope = kv.clone(), k_rope.clone()
        if where == "rope":
            rope[at] = value
        else:
            bad[at, :, :NOPE] = value if where == "keys" else bad[at, :, :NOPE]
            bad[at, :, NOPE:] = value if where == "values" else bad[at, :, NOPE:]
        got, lse = latent_prefill(*args(bad, rope))
        keep = list(range(at)) + list(range(300, 637))
        assert torch.equal(got[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep]), where
        if math.isnan(value):
            assert bool(got[at:300].isnan().all()), where
    bad = kv.clone()
    bad[377:] = value  # the last sequence's rows: those before it end inside a tile
    got, _ = latent_prefill(*args(bad, k_rope))
    assert torch.equal(got[:377], want[:377])


def test_prefill_takes_any_strides():
    from gemq_b200.kernels import latent_prefill
    parts = [(200, 260), (40, 40)]
    q, kv, k_rope, cu_q, cu_k = prefill_case(parts, 4, torch.float16)
    want = latent_prefill(q[..., :NOPE].contiguous(), q[..., NOPE:].contiguous(), kv, k_rope, cu_q, cu_k, 0.07)
    wide = torch.full((300, 704), NAN, dtype=torch.float16, device="cuda")  # keys inside the rows of another projection
    wide[:, 512:576] = k_rope
    heads_first = kv.transpose(0, 1).contiguous().transpose(0, 1)
    got = latent_prefill(q[..., :NOPE], q[..., NOPE:], heads_first, wide[:, 512:576], cu_q, cu_k, 0.07)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_prefill_reports_bad_offsets():
    from gemq_b200.kernels import latent_error, latent_prefill
    parts = [(100, 100), (60, 80)]
    q, kv, k_rope, cu_q, cu_k = prefill_case(parts, 2, torch.bfloat16)
    for cq, ck in (([0, 100, 160], [0, 100, 10 ** 6]), ([0, 100, 160], [-50, 100, 180]), ([0, 100, 160], [0, 200, 180]),
                   ([0, 100, 999], [0, 100, 180]), ([-3, 100, 160], [0, 100, 180]), ([0, 170, 160], [0, 100, 180])):
        cq, ck = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (cq, ck))
        latent_prefill(q[..., :NOPE], q[..., NOPE:], kv, k_rope, cq, ck, 0.07)
        assert latent_error() == 42


# ---- rows into the cache ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,R,page", [(1, 16, 512, 64), (7, 5, 512, 16), (40, 0, 128, 32), (333, 16, 384, 64), (2000, 1, 256, 128)])
def test_append(T, H, R, page, dtype):
    from gemq_b200.kernels import latent_append
    gen = generator(T)
    wide = (3 * torch.randn(T, R + ROPE + 24, device="cuda", generator=gen)).to(dtype)
    kv = wide[:, 8:8 + R + ROPE]  # inside the rows of a joint projection
    q = torch.randn(T, H, NOPE + ROPE, device="cuda", generator=gen).to(dtype)
    w = (1 + 0.3 * torch.randn(R, device="cuda", generator=gen)).to(dtype)
    inv = 1.0 / 1e4 ** (torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float32) / ROPE)
    pos = torch.randint(0, 160000, (T,), device="cuda", generator=gen)
    pages = -(-T // page) + 2
    cache = torch.randn(pages, page, R + ROPE, device="cuda", generator=gen).to(dtype)
    before = cache.clone()
    slots = torch.randperm(pages * page, device="cuda", generator=gen)[:T]
    slots[T // 2::5] = -1
    q_out, rows = latent_append(kv, q[..., NOPE:], w, 1e-6, inv, pos, slots, cache, 1.25)
    x = kv.double()
    turn = torch.polar(torch.tensor(1.25, dtype=torch.float64, device="cuda"), pos.double()[:, None] * inv.double())

    def rot(v, t):
        return torch.view_as_real(torch.view_as_complex(v.unflatten(-1, (-1, 2)).contiguous()) * t).flatten(-2)

    want = torch.cat([x[:, :R] * torch.rsqrt(x[:, :R].square().mean(1, keepdim=True) + 1e-6) * w.double(), rot(x[:, R:], turn)], 1)
    # one rounding, and 32-bit errors: of the mean (512 terms in a tree) and its root, of the products, of sine and cosine; below the
    # normal numbers (fp16: 2^-14) the type's steps are eps * tiny apart whatever the value, and a rounding is off by half of one
    step, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).eps * torch.finfo(dtype).tiny / 2
    size = torch.cat([want[:, :R].abs(), 1.25 * x[:, R:].abs().unflatten(-1, (-1, 2)).sum(-1).repeat_interleave(2, -1)], 1)
    assert bool(((rows.double() - want).abs() <= step * want.abs() + 2.0 ** -20 * size + least).all())
    if H:
        qx = q[..., NOPE:].double()
        want_q = rot(qx, turn[:, None])
        size = 1.25 * qx.abs().unflatten(-1, (-1, 2)).sum(-1).repeat_interleave(2, -1)
        assert bool(((q_out.double() - want_q).abs() <= step * want_q.abs() + 2.0 ** -20 * size + least).all())
    assert q_out.shape == (T, H, ROPE)
    kept = slots >= 0
    flat = before.view(-1, R + ROPE)
    flat[slots[kept]] = rows[kept]
    assert torch.equal(cache, before)  # the rows as they were returned, every other row as it was


def test_append_reports_bad_slots():
    from gemq_b200.kernels import latent_append, latent_error
    kv, w = torch.ones(4, 576, dtype=torch.float16, device="cuda"), torch.ones(512, dtype=torch.float16, device="cuda")
    cache = torch.zeros(2, 64, 576, dtype=torch.float16, device="cuda")
    inv, pos = torch.ones(32, device="cuda"), torch.arange(4, device="cuda")
    for bad in (128, -2, 2 ** 62, -2 ** 62):
        cache.zero_()
        latent_append(kv, kv[:, None, :64], w, 1e-6, inv, pos, torch.tensor([0, bad, 127, -1], device="cuda"), cache)
        assert latent_error() == 43
        assert cache.view(-1, 576).any(1).nonzero().flatten().tolist() == [0, 127]


# ---- pages --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layers,pages,page,width,dtype", [(1, 9, 16, 192, torch.float16), (27, 12, 64, 576, torch.bfloat16),
                                                           (3, 7, 1, 8, torch.float16), (2, 300, 3, 5, torch.float64), (2, 5, 7, 16, torch.uint8)])
def test_copy_pages(layers, pages, page, width, dtype):
    from gemq_b200.kernels import copy_pages, latent_error
    gen = generator(pages)
    big = torch.randint(0, 100, (layers, pages, 2, page, width), device="cuda", generator=gen).to(dtype)
    cache = big[:, :, 1]  # every other page of a larger buffer
    if page * width * big.element_size() % 16:
        with pytest.raises(ValueError, match="16 bytes"):
            copy_pages(cache, torch.zeros(1, dtype=torch.int64, device="cuda"), torch.ones(1, dtype=torch.int64, device="cuda"))
        return
    perm = torch.randperm(pages, device="cuda", generator=gen)
    n = pages // 2
    src, dst = perm[:n].clone(), perm[n:2 * n].clone()
    src[0] = src[-1]  # a page may be copied to several places
    dst[1:2] = src[1:2]  # onto itself: left alone
    want = big.clone()
    want[:, :, 1].index_copy_(1, dst, big[:, :, 1].index_select(1, src))
    copy_pages(cache, src, dst)
    assert torch.equal(big, want)
    if layers == 1:
        copy_pages(cache[0], dst[-1:], dst[-1:])
        assert torch.equal(big, want)
    for bad in (pages, -1, 2 ** 60):
        copy_pages(cache, torch.tensor([0, bad], device="cuda"), torch.tensor([bad, 1], device="cuda"))
        assert latent_error() == 41 and torch.equal(big, want)
    copy_pages(cache, src[:0], dst[:0])


# ---- what others in the same tile hold ------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_numbers_of_others_change_no_bit_of_decode(dtype):
    """Pieces of several tiles, so that the reference of a row's weights may move behind the first: a large finite row that only the later queries see,
    and a large query of one head, leave every other query bit for bit what it was."""
    from gemq_b200.kernels import latent_decode
    lens = [400 + 7 * i % 200 for i in range(300)]
    q_latent, q_rope, cache, table, n, rows = decode_case(lens, 4, 16, 512, 64, dtype, seed=1)
    want = latent_decode(q_latent, q_rope, cache, table, n, 192 ** -0.5)
    bad = cache.clone()
    for b, (pages, length) in enumerate(rows):  # seen by queries 2 and 3
        bad[pages[(length - 2) // 64], (length - 2) % 64] = 60 * torch.cat([q_latent[b, 3, 5], q_rope[b, 3, 5]])
    assert bool(bad[rows[0][0][0]].isfinite().all())
    got = latent_decode(q_latent, q_rope, bad, table, n, 192 ** -0.5)
    assert not torch.equal(got[0][:, 2:], want[0][:, 2:])
    assert all(torch.equal(a[:, :2], b[:, :2]) for a, b in zip(got, want))
    large = q_latent.clone()
    large[:, :, 5] *= 64
    got = latent_decode(large, q_rope, cache, table, n, 192 ** -0.5)
    others = [h for h in range(16) if h != 5]
    assert all(torch.equal(a[:, :, others], b[:, :, others]) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_queries_of_others_change_no_bit_behind_a_prefix(dtype):
    """Rows of several sequences stand in one tile of queries: a large one is its own sequence's."""
    from gemq_b200.kernels import latent_decode_shared
    B = 40
    q_latent, q_rope, cache, table, n, _ = decode_case([30] * B + [40000], 1, 16, 512, 64, dtype, seed=2)
    args = (q_rope[:B], cache, table[:B].contiguous(), n[:B].contiguous(), table[B:].contiguous(), n[B:].contiguous(),
            torch.tensor([0, B], dtype=torch.int32, device="cuda"), 192 ** -0.5)
    want = latent_decode_shared(q_latent[:B], *args)
    large = q_latent[:B].clone()
    large[::4] *= 64
    got = latent_decode_shared(large, *args)
    keep = [b for b in range(B) if b % 4]
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", [140, 200, 270])
def test_large_numbers_of_others_change_no_bit_of_prefill(at, dtype):
    """A large finite key in a tile behind the first, and a large query, beside queries of the same warp."""
    from gemq_b200.kernels import latent_prefill
    q, kv, k_rope, cu_q, cu_k = prefill_case([(300, 300), (40, 340)], 16, dtype)
    args = lambda q, kv: (q[..., :NOPE], q[..., NOPE:], kv, k_rope, cu_q, cu_k, 192 ** -0.5)  # noqa: E731
    want = latent_prefill(*args(q, kv))
    bad = kv.clone()
    bad[at, :, :NOPE] = 60 * q[at + 10, :, :NOPE]  # aligned with a later query of the tile
    assert bool(bad.isfinite().all())
    got = latent_prefill(*args(q, bad))
    assert not torch.equal(got[0][at:300], want[0][at:300])
    keep = list(range(at)) + list(range(300, 340))
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, want))
    large = q.clone()
    large[at] *= 64
    large[320] *= 64
    got = latent_prefill(*args(large, kv))
    keep = [i for i in range(340) if i not in (at, 320)]
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, want))


@pytest.mark.parametrize("B,G,pitch", [(4, 6, 3), (40, 7, 40), (512, 600, 20000)])
def test_decode_shared_of_starts_that_go_back(B, G, pitch):
    """Starts by which every other group has the whole batch: reported, and all results are NaN.  (The last of them asks for more than 2^31 quarters
    of a tile.)"""
    from gemq_b200.kernels import latent_decode_shared, latent_error
    q_latent, q_rope, cache, table, n, _ = decode_case([1 + 9 * i % 80 for i in range(B)], 1, 16, 512, 64, torch.bfloat16)
    prefix = torch.zeros(G, pitch, dtype=torch.int32, device="cuda")
    full, none = torch.full((G,), 64 * pitch, dtype=torch.int32, device="cuda"), torch.zeros(G, dtype=torch.int32, device="cuda")
    run = lambda lens, starts: latent_decode_shared(q_latent, q_rope, cache, table, n, prefix, lens,  # noqa: E731
                                                    torch.tensor(starts, dtype=torch.int32, device="cuda"), 0.07)
    run(none, [0] + [B] * G)
    assert latent_error() == 0
    for starts in ([B * (g % 2) for g in range(G)] + [B], [0] + [B + 1] * G, [-1] + [B] * G, [0] * (G + 1), [B] * (G + 1), [0] + [2 ** 31 - 1, -2 ** 31] * (G // 2) + [B] * (G % 2)):
        got = run(full, starts)
        assert latent_error() == 42
        assert all(bool(t.isnan().all()) for t in got), starts


def test_decode_shared_without_a_prefix_page():
    """A prefix table without columns: the sequences' own rows are all there is."""
    from gemq_b200.kernels import latent_decode_shared
    q_latent, q_rope, cache, table, n, rows = decode_case([100, 30, 0], 2, 16, 512, 64, torch.float16)
    none, starts = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda")
    got = latent_decode_shared(q_latent, q_rope, cache, table, n, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), none, starts, 0.07)
    check_decode(*got, q_latent, q_rope, [rows_of(cache, r) for r in rows], 0.07)
    same = latent_decode_shared(q_latent, q_rope, cache, table, n, torch.zeros(2, 5, dtype=torch.int32, device="cuda"), none, starts, 0.07)
    assert all(torch.equal(a, b) for a, b in zip(got, same))


# ---- what is reported ---------------------------------------------------------------------------------
def test_errors_are_the_latent_operators_own():
    """A code that the linears' waits left in their word is neither returned nor cleared."""
    from gemq_b200.kernels import copy_pages, latent_error
    from gemq_b200.kernels._runtime import error_word
    word = error_word(torch.device("cuda", torch.cuda.current_device()))
    assert int(word.item()) == 0
    try:
        word.fill_(7)
        assert latent_error() == 0 and int(word.item()) == 7
        copy_pages(torch.zeros(2, 4, 2, 8, device="cuda"), torch.tensor([9], device="cuda"), torch.tensor([1], device="cuda"))
        assert int(word.item()) == 7 and latent_error("cuda") == 41 and latent_error() == 0
    finally:
        word.zero_()


def test_errors_of_other_streams_are_waited_for():
    from gemq_b200.kernels import copy_pages, latent_error
    cache, src, dst = torch.zeros(2, 4, 2, 8, device="cuda"), torch.tensor([9], device="cuda"), torch.tensor([1], device="cuda")
    side = torch.cuda.Stream()
    for _ in range(3):  # the first loads the kernels, which waits by itself
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)  # a tenth of a second
            copy_pages(cache, src, dst)
        assert latent_error() == 41 and latent_error() == 0


# ---- writes into the cache ------------------------------------------------------------------------------
def test_writes_into_the_cache_are_seen_by_autograd():
    """What a differentiable product has kept of the cache, and an operator then overwrote, is not used for a gradient."""
    from gemq_b200.kernels import copy_pages, latent_append
    cache = torch.ones(2, 64, 576, dtype=torch.float16, device="cuda")
    kv, w, i64 = torch.ones(1, 576, dtype=torch.float16, device="cuda"), torch.ones(512, dtype=torch.float16, device="cuda"), torch.int64
    slot, page = torch.zeros(1, dtype=i64, device="cuda"), torch.ones(1, dtype=i64, device="cuda")
    append = lambda c: latent_append(kv, kv[:, None, :64], w, 1e-6, torch.ones(32, device="cuda"), slot, slot, c)  # noqa: E731
    for name, write in (("native", append), ("no heads", lambda c: latent_append(kv, kv[:, None, :64][:, :0], w, 1e-6, torch.ones(32, device="cuda"), slot, slot, c)),
                        ("by name", lambda c: latent_append(kv, kv[:, None, :64], w, 1e-6, torch.ones(32, device="cuda"), slot, slot, cache=c)),
                        ("one layer", lambda c: copy_pages(c, slot, page)), ("layers", lambda c: copy_pages(c.view(1, 2, 64, 576), slot, page)),
                        ("pages by name", lambda c: copy_pages(src=slot, dst=page, cache=c))):
        before = cache._version
        write(cache)
        assert cache._version > before, name
        x = torch.ones(576, dtype=torch.float16, device="cuda", requires_grad=True)
        y = (cache[0] * x).sum()
        write(cache)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        c = torch.ones(2, 64, 576, dtype=torch.float16, device="cuda")
        append(c)
        copy_pages(c, slot, page)
        assert torch.equal(c[0], c[1])


@pytest.mark.parametrize("native", [True, False])
def test_copy_pages_of_one_layer(native):
    """The forms without a dimension for the layers, pages further apart than they are long; four dimensions beside them, in both routes."""
    from gemq_b200.kernels import copy_pages
    gen = generator(5)
    src, dst = torch.tensor([4, 0, 4, 8], device="cuda"), torch.tensor([1, 2, 7, 8], device="cuda")
    for big, view in ((torch.randn(9, 3, 4, 24, device="cuda", generator=gen), lambda t: t[:, 1]),      # [9, 4, 24], 288 apart
                      (torch.randn(9, 40, device="cuda", generator=gen), lambda t: t[:, 8:28]),          # [9, 20], 40 apart
                      (torch.randn(18, 8, 16, device="cuda", generator=gen).half(), lambda t: t[::2]),
                      (torch.randn(3, 9, 2, 5, 8, device="cuda", generator=gen), lambda t: t[:, :, 1]),  # layers
                      (torch.randn(9, 3, 5, 8, device="cuda", generator=gen), lambda t: t.transpose(0, 1))):
        want = big.clone()
        dim = 1 if view(big).dim() >= 4 else 0
        view(want).index_copy_(dim, dst, view(big).index_select(dim, src))
        if native:
            copy_pages(view(big), src, dst)
        else:
            torch.ops.gemq_b200.copy_pages(view(big), src, dst)
        assert torch.equal(big, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix,sizes,own,S,H,R,page", [
    ([200], [3], [1, 64, 100], 1, 5, 512, 64),          # 15 rows in the batch
    ([90, 0], [1, 1], [30, 7], 2, 4, 256, 16),          # 16
    ([1000], [4], [1, 0, 40], 1, 8, 512, 32),           # 32
    ([300, 70], [2, 1], [5, 200], 3, 3, 128, 64),       # 27
    ([40000], [2], [1, 100], 1, 16, 512, 64),           # 32, a prefix over all CTAs
])
def test_decode_shared_of_few_rows(prefix, sizes, own, S, H, R, page, dtype):
    test_decode_shared(prefix, sizes, own, S, H, R, page, dtype)


@pytest.mark.parametrize("lens,S,H,page", [([131072], 1, 16, 64), ([131071, 3, 131072], 2, 16, 16), ([200001, 70], 1, 64, 128)])
def test_decode_of_far_positions(lens, S, H, page):
    test_decode(lens, S, H, 512, page, torch.bfloat16)
