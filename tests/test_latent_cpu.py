"""Latent operators without a GPU: registration, what they refuse, and the cache's bookkeeping."""
import ctypes as C
import random

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from gemq_b200 import _capi
from gemq_b200 import kernels as K
from gemq_b200.kernels import latent_attention as L

B, S, H, R = 3, 2, 5, 256
f16, bf16, i32, i64 = torch.float16, torch.bfloat16, torch.int32, torch.int64


def decode_args(**over):
    a = dict(q_latent=torch.zeros(B, S, H, R, dtype=f16), q_rope=torch.zeros(B, S, H, 64, dtype=f16), cache=torch.zeros(7, 64, R + 64, dtype=f16),
             table=torch.zeros(B, 4, dtype=i32), lens=torch.zeros(B, dtype=i32))
    return {**a, **over}


def shared_args(**over):
    a = decode_args(prefix_table=torch.zeros(2, 3, dtype=i32), prefix_lens=torch.zeros(2, dtype=i32), starts=torch.zeros(3, dtype=i32))
    return {**a, **over}


def prefill_args(**over):
    a = dict(q_nope=torch.zeros(9, H, 128, dtype=f16), q_rope=torch.zeros(9, H, 64, dtype=f16), kv=torch.zeros(11, H, 256, dtype=f16),
             k_rope=torch.zeros(11, 64, dtype=f16), cu_q=torch.zeros(3, dtype=i32), cu_k=torch.zeros(3, dtype=i32))
    return {**a, **over}


def append_args(**over):
    a = dict(kv=torch.zeros(6, R + 64, dtype=f16), q_rope=torch.zeros(6, H, 64, dtype=f16), norm_weight=torch.zeros(R, dtype=f16), eps=1e-6,
             inv_freq=torch.zeros(32), positions=torch.zeros(6, dtype=i64), slots=torch.zeros(6, dtype=i64), cache=torch.zeros(7, 64, R + 64, dtype=f16))
    return {**a, **over}


def test_operators_are_registered_with_their_shapes():
    for name in ("latent_append", "latent_decode", "latent_decode_shared", "latent_prefill", "copy_pages"):
        assert hasattr(torch.ops.gemq_b200, name), name
    with FakeTensorMode():
        for args in (decode_args(), shared_args()):
            f = K.latent_decode if "starts" not in args else K.latent_decode_shared
            out, lse = f(*args.values(), 0.1)
            assert out.shape == (B, S, H, R) and out.dtype == f16 and lse.shape == (B, S, H) and lse.dtype == torch.float32
        out, lse = K.latent_prefill(*prefill_args().values(), 0.1)
        assert out.shape == (9, H, 128) and out.dtype == f16 and lse.shape == (9, H) and lse.dtype == torch.float32
        q, rows = K.latent_append(*append_args().values())
        assert q.shape == (6, H, 64) and rows.shape == (6, R + 64)


def test_operators_refuse_cpu_tensors_and_gradients():
    for f, args in ((K.latent_decode, decode_args()), (K.latent_decode_shared, shared_args()), (K.latent_prefill, prefill_args())):
        with pytest.raises(RuntimeError, match="CUDA"):
            f(*args.values(), 0.1)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.latent_append(*append_args().values())
    with pytest.raises(RuntimeError, match="CUDA"):
        K.copy_pages(torch.zeros(2, 3, 4, 8), torch.zeros(1, dtype=i64), torch.ones(1, dtype=i64))


NARROW = torch.zeros(B, S, H, R + 8, dtype=f16)[..., 4:R + 4]  # rows 8 bytes off a 16-byte boundary
BAD = [
    (L.latent_decode, decode_args, dict(cache=torch.zeros(7, 48, R + 64, dtype=f16)), "page size"),
    (L.latent_decode, decode_args, dict(cache=torch.zeros(7, 0, R + 64, dtype=f16)), "page size"),
    (L.latent_decode, decode_args, dict(cache=torch.zeros(7, 64, 200 + 64, dtype=f16)), "rank"),
    (L.latent_decode, decode_args, dict(cache=torch.zeros(7, 64, R + 64, dtype=bf16)), "cache must be"),
    (L.latent_decode, decode_args, dict(cache=torch.zeros(0, 64, R + 64, dtype=f16)), "rows"),
    (L.latent_decode, decode_args, dict(cache=torch.zeros(7, 64, R + 128, dtype=f16)[..., :R + 64]), "one behind the other"),
    (L.latent_decode, decode_args, dict(cache=torch.zeros(1, 64, R + 64, dtype=f16).expand(7, -1, -1)), "pages apart"),
    (L.latent_decode, decode_args, dict(q_latent=torch.zeros(B, S, H, 128, dtype=f16)), "q_latent"),
    (L.latent_decode, decode_args, dict(q_latent=torch.zeros(B, 0, H, R, dtype=f16), q_rope=torch.zeros(B, 0, H, 64, dtype=f16)), "a step and a head"),
    (L.latent_decode, decode_args, dict(q_latent=NARROW), "16-byte"),
    (L.latent_decode, decode_args, dict(q_rope=torch.zeros(B, S, H, 64, dtype=bf16)), "q_rope"),
    (L.latent_decode, decode_args, dict(table=torch.zeros(B, 4, dtype=i64)), "table"),
    (L.latent_decode, decode_args, dict(table=torch.zeros(B + 1, 4, dtype=i32)), "table"),
    (L.latent_decode, decode_args, dict(table=torch.zeros(4, B, dtype=i32).t()), "table"),
    (L.latent_decode, decode_args, dict(lens=torch.zeros(B, 1, dtype=i32)), "lens"),
    (L.latent_decode_shared, shared_args, dict(starts=torch.zeros(2, dtype=i32)), "starts"),
    (L.latent_decode_shared, shared_args, dict(prefix_lens=torch.zeros(2, dtype=i64)), "prefix_lens"),
    (L.latent_decode_shared, shared_args, dict(prefix_table=torch.zeros(0, 3, dtype=i32)), "prefix_table"),
    (L.latent_prefill, prefill_args, dict(q_nope=torch.zeros(9, H, 64, dtype=f16)), "q_nope"),
    (L.latent_prefill, prefill_args, dict(q_nope=torch.zeros(9, H, 128)), "fp16 or bf16"),
    (L.latent_prefill, prefill_args, dict(kv=torch.zeros(11, H + 1, 256, dtype=f16)), "kv must"),
    (L.latent_prefill, prefill_args, dict(k_rope=torch.zeros(10, 64, dtype=f16)), "k_rope"),
    (L.latent_prefill, prefill_args, dict(kv=torch.zeros(11, H, 256, dtype=bf16)), "one type"),
    (L.latent_prefill, prefill_args, dict(cu_k=torch.zeros(4, dtype=i32)), "cu_k"),
    (L.latent_prefill, prefill_args, dict(cu_q=torch.zeros(0, dtype=i32)), "cu_q"),
    (L.latent_append, append_args, dict(norm_weight=torch.zeros(R)), "norm_weight"),
    (L.latent_append, append_args, dict(kv=torch.zeros(6, R, dtype=f16)), "kv must"),
    (L.latent_append, append_args, dict(inv_freq=torch.zeros(64)), "inv_freq"),
    (L.latent_append, append_args, dict(slots=torch.zeros(6, dtype=i32)), "slots"),
    (L.latent_append, append_args, dict(positions=torch.zeros(5, dtype=i64)), "positions"),
]


@pytest.mark.parametrize("f,base,over,match", BAD)
def test_refusals(f, base, over, match, monkeypatch):
    """With the question of the device left out: what is wrong is named before anything is launched."""
    monkeypatch.setattr(L, "require_cuda", lambda *t: t[0].device)
    scale = () if f is L.latent_append else (0.1,)
    with pytest.raises(ValueError, match=match):
        f._init_fn(*base(**over).values(), *scale)


def test_copy_pages_refusals(monkeypatch):
    monkeypatch.setattr(L, "require_cuda", lambda *t: t[0].device)
    one = torch.zeros(1, dtype=i64)
    for cache, src, dst, match in ((torch.zeros(4, 3, 2, 2, dtype=f16), one, one, "16 bytes"),
                                   (torch.zeros(4, 3, 8, 16, dtype=f16).transpose(2, 3), one, one, "contiguous"),
                                   (torch.zeros(4, 3, 2, 8, dtype=f16), one.int(), one, "src"),
                                   (torch.zeros(4, 3, 2, 8, dtype=f16), one, torch.zeros(2, dtype=i64), "dst"),
                                   (torch.zeros(4, 0, 2, 8, dtype=f16), one, one, "empty")):
        with pytest.raises(ValueError, match=match):
            L.copy_pages._init_fn(cache, src, dst)
    L.copy_pages._init_fn(torch.zeros(4, 3, 2, 8, dtype=f16), one[:0], one[:0])


def test_library_refuses():
    """The C entries: every refusal comes before the device is touched (there is none here)."""
    A = _capi.LatentDecode()
    assert _capi.lib.gemq_latent_decode(C.byref(A), None, 0, None) == -1
    p = 1 << 20
    ok = dict(q_latent=p, q_rope=p, cache=p, table=p, lens=p, out=p, lse=p, err=p, batch=2, steps=1, heads=3, rank=512, n_pages=5, page_size=64,
              table_pitch=4, page_stride=64 * 576)

    def code(**over):
        A = _capi.LatentDecode()
        for k, v in {**ok, **over}.items():
            setattr(A, k, v)
        return _capi.lib.gemq_latent_decode(C.byref(A), None, 0, None)

    assert code() == -3  # no workspace
    for over, want in ((dict(rank=192), -2), (dict(rank=1024), -2), (dict(page_size=8), -2), (dict(page_size=96), -2), (dict(heads=0), -1),
                       (dict(out=None), -1), (dict(q_latent=p + 8), -5), (dict(page_stride=4), -5), (dict(page_stride=0), -2), (dict(groups=1), -1),
                       (dict(batch=1 << 20, steps=1 << 10, heads=128), -2), (dict(table_pitch=1 << 30), -2), (dict(batch=-1), -1)):
        assert code(**over) == want, over
    assert code(batch=0) == 0
    A = _capi.LatentPrefill()
    A.q_rows = 4
    assert _capi.lib.gemq_latent_prefill(C.byref(A), None) == -1
    A.q_rows = 0
    assert _capi.lib.gemq_latent_prefill(C.byref(A), None) == 0
    for k, v in dict(q_nope=p, q_rope=p, kv=p, k_rope=p, cu_q=p, cu_k=p, out=p, lse=p, err=p, batch=1, q_rows=4, k_rows=4, heads=2,
                     k_rope_stride=64).items():
        setattr(A, k, v)
    A.q_nope_stride[:], A.q_rope_stride[:], A.kv_stride[:] = (256, 128), (128, 64), (512, 0)
    assert _capi.lib.gemq_latent_prefill(C.byref(A), None) == -2  # a stride of 0
    A.kv_stride[:] = (512, 4)
    assert _capi.lib.gemq_latent_prefill(C.byref(A), None) == -5
    f = _capi.lib.gemq_latent_append
    assert f(p, 576, p, 64, 64, p, 1e-6, p, 1.0, p, p, p, 64 * 576, 5, 64, p, p, 3, 2, 500, 0, p, None) == -2
    assert f(p, 576, p, 64, 64, p, 1e-6, p, 1.0, p, None, p, 64 * 576, 5, 64, p, p, 3, 2, 512, 0, p, None) == -1
    assert f(p, 577, p, 64, 64, p, 1e-6, p, 1.0, p, p, p, 64 * 576, 5, 64, p, p, 3, 2, 512, 0, p, None) == -5
    assert f(p, 576, p, 64, 64, p, 1e-6, p, 1.0, p, p, p, 64 * 576, 5, 64, p, p, 0, 2, 512, 0, p, None) == 0
    g = _capi.lib.gemq_copy_pages
    assert g(p, 0, 24, 1, 4, 16, p, p, 1, p, None) == -5 and g(p, 0, 32, 1, 4, 0, p, p, 1, p, None) == -1 and g(p, 0, 32, 1, 4, 16, p, p, 0, p, None) == 0


# ---- the cache ----------------------------------------------------------------------------------------
@pytest.fixture
def cache(monkeypatch):
    from gemq_b200.inference import latent_cache as M
    monkeypatch.setattr(M, "copy_pages", lambda c, src, dst: c.index_copy_(1, dst, c.index_select(1, src)))
    return M.PagedLatentCache(2, 12, page_size=16, rank=128, device="cpu")


def write(cache, plan, values):
    cache.pages.view(2, -1, 192)[:, plan.slots] = values[None, :, None].to(cache.pages.dtype).expand(2, -1, 192)


def read(cache, seq):
    n = cache.length(seq)
    return cache.pages[:, cache.pages_of(seq)].flatten(1, 2)[:, :n, 0].float()


def test_cache_keeps_what_each_sequence_wrote(cache):
    """Any order of extending, forking, cutting, freeing and compacting: every sequence reads what was written to it, no page has two
    owners that write, the free pages are those that nobody has."""
    rng, held, count = random.Random(3), {}, 0
    shared = 0
    for step in range(600):
        do = rng.choice(("new", "extend", "extend", "extend", "fork", "free", "truncate", "compact"))
        seq = rng.choice(sorted(held)) if held else None
        try:
            if do == "new":
                held[cache.new()] = []
            elif seq is None:
                continue
            elif do == "extend":
                n = rng.randint(0, 20)
                plan = cache.plan_prefill([seq], [n])
                values = torch.arange(count, count + n) % 256  # exact in 16 bits
                count += n
                assert plan.positions.tolist() == list(range(len(held[seq]), len(held[seq]) + n))
                write(cache, plan, values)
                held[seq] = held[seq] + values.tolist()
            elif do == "fork":
                held[cache.fork(seq)] = list(held[seq])
            elif do == "free":
                cache.free(seq)
                del held[seq]
            elif do == "truncate":
                n = rng.randint(0, len(held[seq]))
                cache.truncate(seq, n)
                held[seq] = held[seq][:n]
            else:
                before = cache.free_pages
                cache.compact()
                assert cache.free_pages == before
                assert {p for s in held for p in cache.pages_of(s)} == set(range(12 - before))
        except RuntimeError as e:
            assert "full" in str(e)
        for s, want in held.items():
            got = read(cache, s)
            assert cache.length(s) == len(want) and got.tolist() == [want, want], (step, do)
        users = [sum(p in cache.pages_of(s) for s in held) for p in range(12)]
        assert cache.free_pages == users.count(0) and cache._users == users
        shared = max(shared, max(users))
        if rng.random() < 0.1 and held:
            cache.free(sorted(held)[0])
            del held[sorted(held)[0]]
    assert shared > 1


def test_cache_plans(cache):
    a = cache.new()
    plan = cache.plan_prefill([a], [35])
    assert plan.cu_q.tolist() == [0, 35] and plan.cu_k.tolist() == [0, 35] and plan.rows is None and plan.steps == 0
    b = cache.fork(a)
    assert cache.pages_of(b)[:2] == cache.pages_of(a)[:2] and cache.pages_of(b)[2] != cache.pages_of(a)[2]
    c = cache.new()
    plan = cache.plan_prefill([b, c], [2, 17])
    assert plan.cu_q.tolist() == [0, 2, 19] and plan.cu_k.tolist() == [0, 37, 54] and plan.lens.tolist() == [37, 17]
    assert plan.rows[:32].tolist() == [p * 16 + i for p in cache.pages_of(a)[:2] for i in range(16)] and plan.rows.numel() == 54
    plan = cache.plan_decode([a, b, c], 2, groups=[2, 1])
    assert plan.positions.tolist() == [35, 36, 37, 38, 17, 18] and plan.starts.tolist() == [0, 2, 3]
    assert plan.prefix_lens.tolist() == [32, 0] and plan.prefix_table[0, :2].tolist() == cache.pages_of(a)[:2]
    assert plan.lens.tolist() == [5, 7, 19] and plan.table[0, 0].item() == cache.pages_of(a)[2] and plan.table[2, :2].tolist() == cache.pages_of(c)
    plan = cache.plan_decode([a, c])
    assert plan.lens.tolist() == [38, 20] and plan.starts is None and plan.table.dtype == i32 and plan.slots.dtype == i64


def test_cache_refuses(cache):
    from gemq_b200.inference import PagedLatentCache
    a, b = cache.new(), cache.new()
    with pytest.raises(RuntimeError, match="full"):
        cache.extend([a, b], [100, 100])
    assert cache.free_pages == 12 and cache.length(a) == 0  # all or nothing
    for call in (lambda: cache.extend([a, a], [1, 1]), lambda: cache.extend([a], [-1]), lambda: cache.extend([a], [1, 2]),
                 lambda: cache.truncate(a, 1), lambda: cache.plan_decode([a, b], groups=[1]), lambda: cache.plan_decode([a, b], groups=[2, 0]),
                 lambda: PagedLatentCache(1, 4, page_size=24), lambda: PagedLatentCache(1, 0), lambda: PagedLatentCache(1, 4, rank=200),
                 lambda: PagedLatentCache(1, 4, dtype=torch.float32)):
        with pytest.raises(ValueError):
            call()
    cache.free(a)
    with pytest.raises(KeyError):
        cache.free(a)
    with pytest.raises(KeyError):
        cache.fork(a)


def test_attention_layer_refuses():
    from types import SimpleNamespace
    from gemq_b200.inference import LatentAttention
    lin = lambda o, i: torch.nn.Linear(i, o, bias=False)  # noqa: E731
    with pytest.raises(ValueError, match="kv_b_proj"):
        LatentAttention(lin(768, 32), lin(192, 32), torch.ones(128), 1e-6, lin(1000, 128), lin(32, 512), 4, torch.ones(32))
    with pytest.raises(ValueError, match="bias"):
        LatentAttention(lin(768, 32), lin(192, 32), torch.ones(128), 1e-6, torch.nn.Linear(128, 1024), lin(32, 512), 4, torch.ones(32))
    with pytest.raises(ValueError, match="inv_freq"):
        LatentAttention(lin(768, 32), lin(192, 32), torch.ones(128), 1e-6, lin(1024, 128), lin(32, 512), 4, torch.ones(64))
    cfg = SimpleNamespace(qk_nope_head_dim=128, qk_rope_head_dim=64, v_head_dim=128, rope_scaling={"type": "yarn"}, num_attention_heads=4)
    with pytest.raises(ValueError, match="rotation"):
        LatentAttention.from_hf(cfg, None)
    cfg.v_head_dim = 64
    with pytest.raises(ValueError, match="128"):
        LatentAttention.from_hf(cfg, None)


def test_attention_layer_follows_its_weights():
    """The halves that the absorbed form reads are those of the weight that was loaded; the frequencies stay in 32 bits."""
    from gemq_b200.inference import LatentAttention
    make = lambda: LatentAttention(*(torch.nn.Linear(i, o, bias=False) for i, o in ((32, 768), (32, 192))), torch.rand(128), 1e-6,  # noqa: E731
                                   torch.nn.Linear(128, 1024, bias=False), torch.nn.Linear(512, 32, bias=False), 4, torch.rand(32))
    a, b = make(), make()
    assert not torch.equal(a.w_keys, b.w_keys) and not any(k.startswith("w_") for k in a.state_dict())
    a.load_state_dict(b.state_dict())
    w = b.kv_b_proj.weight.view(4, 256, 128)
    assert torch.equal(a.w_keys, w[:, :128]) and torch.equal(a.w_values, w[:, 128:].transpose(1, 2)) and torch.equal(a.norm_weight, b.norm_weight)
    a.half()
    assert a.w_keys.dtype == a.norm_weight.dtype == f16 and a.inv_freq.dtype == torch.float32


def test_taking_an_error_refuses():
    assert _capi.lib.gemq_latent_take_error(None, 1 << 20, None) == -1 and _capi.lib.gemq_latent_take_error(1 << 20, None, None) == -1
    with pytest.raises(ValueError, match="CUDA"):
        K.latent_error("cpu")


def test_a_decode_plan_has_a_step(cache):
    """None would be the plan of a prefill; nothing is taken by a refused one."""
    a = cache.new()
    cache.extend([a], [20])
    for steps in (0, -1):
        with pytest.raises(ValueError, match="step"):
            cache.plan_decode([a], steps)
    assert cache.length(a) == 20 and cache.free_pages == 10


def test_attention_layer_is_saved_whole():
    """Pickled, copied, and still following the weights that are loaded into it."""
    import copy
    import io
    from gemq_b200.inference import LatentAttention
    make = lambda: LatentAttention(*(torch.nn.Linear(i, o, bias=False) for i, o in ((32, 768), (32, 192))), torch.rand(128), 1e-6,  # noqa: E731
                                   torch.nn.Linear(128, 1024, bias=False), torch.nn.Linear(512, 32, bias=False), 4, torch.rand(32))
    a, b = make(), make()
    file = io.BytesIO()
    torch.save(torch.nn.Sequential(a), file)
    file.seek(0)
    for c in (torch.load(file, weights_only=False)[0], copy.deepcopy(a)):
        assert torch.equal(c.w_keys, a.w_keys) and torch.equal(c.inv_freq, a.inv_freq) and c.scale == a.scale
        c.load_state_dict(b.state_dict())
        assert torch.equal(c.w_keys, b.w_keys) and torch.equal(c.w_values, b.w_values) and not torch.equal(a.w_keys, b.w_keys)
