"""The latent operators as a server uses them together: layers over one paged cache, prompts, drafts, forks, shared prefixes, compaction;
captured steps, several streams."""
import pytest
import torch

from latent_reference import NOPE, ROPE, VALUE

pytestmark = pytest.mark.gpu
D, H, RANK = 256, 4, 512


def make_layer(dtype, seed, quantised):
    from gemq_b200 import synth
    from gemq_b200.inference import LatentAttention, QuantLinear
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def linear(out_f, in_f):
        if quantised:
            return QuantLinear(synth.make_linear(out_f, in_f, 4, 128, gen, "cuda"))
        m = torch.nn.Linear(in_f, out_f, bias=False, device="cuda", dtype=dtype)
        m.weight.data = (torch.randn(out_f, in_f, device="cuda", generator=gen) * in_f ** -0.5).to(dtype)
        return m

    inv = 1.0 / 1e4 ** (torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float32) / ROPE)
    norm = (1 + 0.1 * torch.randn(RANK, device="cuda", generator=gen)).to(dtype)
    return LatentAttention(linear(H * (NOPE + ROPE), D), linear(RANK + ROPE, D), norm, 1e-6, linear(H * (NOPE + VALUE), RANK), linear(D, H * VALUE),
                           H, inv)


def weight(linear):
    from gemq_b200.inference.latent_attention import _weight
    return _weight(linear, torch.float64).detach()


def reference(layer, hidden):
    """One sequence from its first token, in 64 bits, in the expanded form -> [tokens, D]."""
    x = hidden.double()
    n = x.shape[0]
    q = (x @ weight(layer.q_proj).T).view(n, H, NOPE + ROPE)
    c = x @ weight(layer.kv_a_proj).T
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.arange(n, device="cuda").double()[:, None] * layer.inv_freq.double())

    def rot(v, t):
        return torch.view_as_real(torch.view_as_complex(v.unflatten(-1, (-1, 2)).contiguous()) * t).flatten(-2)

    lat = c[:, :RANK] * torch.rsqrt(c[:, :RANK].square().mean(1, keepdim=True) + layer.eps) * layer.norm_weight.double()
    kv = (lat @ weight(layer.kv_b_proj).T).view(n, H, NOPE + VALUE)
    s = torch.einsum("ihd,jhd->hij", q[..., :NOPE], kv[..., :NOPE]) + torch.einsum("ihd,jd->hij", rot(q[..., NOPE:], turn[:, None]), rot(c[:, RANK:], turn))
    s = (s * layer.scale).masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    out = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), kv[..., NOPE:])
    return out.reshape(n, H * VALUE) @ weight(layer.o_proj).T


class Server:
    """Layers with inputs of their own, and what every sequence has been given so far."""

    def __init__(self, dtype, quantised, pages=60, page_size=16):
        from gemq_b200.inference import PagedLatentCache
        self.layers = [make_layer(dtype, i, quantised) for i in range(2)]
        self.cache = PagedLatentCache(2, pages, page_size, RANK, dtype)
        self.gen, self.dtype, self.held = torch.Generator(device="cuda").manual_seed(9), dtype, {}

    def new(self):
        seq = self.cache.new()
        self.held[seq] = torch.zeros(2, 0, D, device="cuda", dtype=self.dtype)
        return seq

    def step(self, seqs, counts, plan):
        x = torch.randn(2, sum(counts), D, device="cuda", generator=self.gen).to(self.dtype)
        at = 0
        for s, n in zip(seqs, counts):
            self.held[s] = torch.cat([self.held[s], x[:, at:at + n]], 1)
            at += n
        eps = torch.finfo(self.dtype).eps
        for i, layer in enumerate(self.layers):
            got = layer(x[i], self.cache, i, plan).double()
            want = torch.cat([reference(layer, self.held[s][i])[-n:] for s, n in zip(seqs, counts) if n])
            # nine roundings of half a step on the way (two of the queries, three of the rows, weights, results, two projections); the five ahead of
            # the scores, which are sums of products of two of them and no larger than 3, move the weights by up to twice 3 times as much
            assert float((got - want).norm() / want.norm()) < (4 + 5 * (1 + 2 * 3)) * eps / 2


@pytest.mark.parametrize("dtype,quantised", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True)])
def test_a_run_of_all_of_them(dtype, quantised):
    from gemq_b200.kernels import latent_error
    s = Server(dtype, quantised)
    a, b, c = s.new(), s.new(), s.new()
    s.step([a, b, c], [70, 1, 33], s.cache.plan_prefill([a, b, c], [70, 1, 33]))
    for steps in (1, 1, 3):
        s.step([a, b, c], [steps] * 3, s.cache.plan_decode([a, b, c], steps))
    s.cache.truncate(a, 74)  # one of the three drafted tokens is kept
    s.held[a] = s.held[a][:, :74]
    d, e = s.cache.fork(a), s.cache.fork(a)
    s.held[d], s.held[e] = s.held[a], s.held[a]
    order = [a, d, e, c, b]
    for steps in (1, 2):
        s.step(order, [steps] * 5, s.cache.plan_decode(order, steps, groups=[3, 2]))
    s.step([e, b], [40, 7], s.cache.plan_prefill([e, b], [40, 7]))  # behind rows that are there
    s.cache.free(c)
    s.cache.free(a)
    assert s.cache.compact() > 0
    s.step([d, b, e], [1] * 3, s.cache.plan_decode([d, b, e]))
    s.step([d, e, b], [1] * 3, s.cache.plan_decode([d, e, b], groups=[2, 1]))
    assert latent_error() == 0


@pytest.mark.parametrize("q_rank", [None, 96])
def test_layer_from_hugging_face(q_rank):
    """The layer made of a Hugging Face module against that module, in 32 bits, over one sequence: a prompt, then tokens one by one."""
    M = pytest.importorskip("transformers.models.deepseek_v2.modeling_deepseek_v2")
    from transformers import DeepseekV2Config
    from gemq_b200.inference import LatentAttention, PagedLatentCache
    cfg = DeepseekV2Config(hidden_size=D, num_attention_heads=H, num_key_value_heads=H, kv_lora_rank=RANK, q_lora_rank=q_rank,
                           qk_nope_head_dim=NOPE, qk_rope_head_dim=ROPE, v_head_dim=VALUE, num_hidden_layers=1, vocab_size=64, intermediate_size=64)
    cfg._attn_implementation = "eager"
    torch.manual_seed(5)
    hf = M.DeepseekV2Attention(cfg, 0).cuda()
    for p in hf.parameters():
        p.data = (p.data + torch.randn_like(p) * (0.1 if p.dim() == 1 else p.shape[1] ** -0.5)).half().float()
    x = torch.randn(1, 50, D, device="cuda").half().float()
    pos = torch.arange(50, device="cuda")[None]
    mask = torch.full((50, 50), float("-inf"), device="cuda").triu(1)[None, None]
    with torch.no_grad():
        want = hf(x, mask, position_embeddings=M.DeepseekV2RotaryEmbedding(cfg).cuda()(x, pos))[0][0]
    layer = LatentAttention.from_hf(cfg, hf.half())
    cache = PagedLatentCache(1, 4, 16, RANK, torch.float16)
    seq = cache.new()
    got = [layer(x[0, :41].half(), cache, 0, cache.plan_prefill([seq], [41]))]
    for i in range(41, 50):
        got.append(layer(x[0, i:i + 1].half(), cache, 0, cache.plan_decode([seq])))
    got = torch.cat(got).float()
    # the roundings of a run's step, and two more where the queries come through a norm
    assert float((got - want).norm() / want.norm()) < (6 + 5 * (1 + 2 * 3)) * torch.finfo(torch.float16).eps / 2


def test_a_decode_step_captured_and_replayed():
    """One graph of both layers' step: plans are copied into its tensors; the pages, the lengths and the rows are those of the replay."""
    from gemq_b200.inference import LatentPlan
    s = Server(torch.float16, False)
    seqs = [s.new(), s.new()]
    s.step(seqs, [50, 5], s.cache.plan_prefill(seqs, [50, 5]))
    x = torch.zeros(2, 2, D, device="cuda", dtype=torch.float16)
    plan = LatentPlan(*(torch.zeros(2, dtype=torch.int64, device="cuda") for _ in range(2)), torch.zeros(2, 8, dtype=torch.int32, device="cuda"),
                      torch.zeros(2, dtype=torch.int32, device="cuda"), 1)
    plan.slots.fill_(-1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for layer in range(2):  # two graphs on one pool of memory
            s.layers[layer](x[layer], s.cache, layer, plan)
        torch.cuda.synchronize()
        for layer in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = s.layers[layer](x[layer], s.cache, layer, plan)
            graphs.append((g, out))
    torch.cuda.synchronize()
    eps = torch.finfo(torch.float16).eps
    for _ in range(12):  # over the end of a page
        now = s.cache.plan_decode(seqs)
        plan.positions.copy_(now.positions)
        plan.slots.copy_(now.slots)
        plan.table[:, :now.table.shape[1]].copy_(now.table)
        plan.lens.copy_(now.lens)
        x.copy_(torch.randn(2, 2, D, device="cuda", generator=s.gen))
        for i, q in enumerate(seqs):
            s.held[q] = torch.cat([s.held[q], x[:, i:i + 1]], 1)
        for layer, (g, out) in enumerate(graphs):
            g.replay()
            want = torch.cat([reference(s.layers[layer], s.held[q][layer])[-1:] for q in seqs])
            assert float((out.double() - want).norm() / want.norm()) < (4 + 5 * (1 + 2 * 3)) * eps / 2


def test_every_operator_captured():
    """Each in a graph of its own, made one after the other and replayed interleaved with eager calls on other data."""
    from gemq_b200 import kernels as K
    gen = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *shape: torch.randn(*shape, device="cuda", generator=gen).half()  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cache, table = r(40, 64, 576), torch.randperm(40, device="cuda", generator=gen).to(torch.int32)[:32].view(2, 16)
    ql, qr, lens = r(2, 1, 16, 512), r(2, 1, 16, 64), i32(900, 70)
    prefix, plens, starts = table[:1, :3].contiguous(), i32(150), i32(0, 2)
    q, kv, kr, cq, ck = r(300, 4, 192), r(300, 4, 256), r(300, 64), i32(0, 100, 300), i32(0, 100, 300)
    rows, w, inv = r(5, 576), r(512), torch.ones(32, device="cuda")
    pos, slots = torch.arange(5, device="cuda"), torch.tensor([2400, -1, 2401, 2402, 2500], device="cuda")
    src, dst = torch.tensor([1, 2], device="cuda"), torch.tensor([38, 39], device="cuda")
    calls = dict(decode=lambda: K.latent_decode(ql, qr, cache, table, lens, 0.07),
                 shared=lambda: K.latent_decode_shared(ql, qr, cache, table, lens, prefix, plens, starts, 0.07),
                 prefill=lambda: K.latent_prefill(q[..., :128], q[..., 128:], kv, kr, cq, ck, 0.07),
                 append=lambda: K.latent_append(rows, qr.expand(2, 5, 16, 64)[0], w, 1e-6, inv, pos, slots, cache),
                 copy=lambda: K.copy_pages(cache, src, dst))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = {}
    with torch.cuda.stream(side):
        for name, call in calls.items():
            call()
        torch.cuda.synchronize()
        for name, call in calls.items():
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                graphs[name] = (call(), g)
    torch.cuda.synchronize()
    for _ in range(3):
        for t in (ql, qr, q, kv, kr, rows):
            t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
        for name in ("append", "copy", "decode", "prefill", "shared"):
            out, g = graphs[name]
            before = cache.clone()
            g.replay()
            after = cache.clone()
            cache.copy_(before)
            want = calls[name]()
            assert torch.equal(cache, after), name
            if out is not None:
                assert all(torch.equal(a, b) for a, b in zip(out, want)), name


def test_calls_on_several_streams_at_once():
    from gemq_b200 import kernels as K
    gen = torch.Generator(device="cuda").manual_seed(4)
    cache = torch.randn(64, 64, 576, device="cuda", generator=gen).half()
    cases = []
    for i in range(4):
        n = [1500 - 300 * i, 64 + i, 900]
        table = torch.randint(0, 64, (3, 24), device="cuda", generator=gen, dtype=torch.int32)
        ql, qr = (torch.randn(3, 1, 16, w, device="cuda", generator=gen).half() for w in (512, 64))
        q, kv = torch.randn(200, 4, 192, device="cuda", generator=gen).half(), torch.randn(260, 4, 256, device="cuda", generator=gen).half()
        cu = [torch.tensor([0, v], dtype=torch.int32, device="cuda") for v in (200, 260)]
        cases.append((ql, qr, table, torch.tensor(n, dtype=torch.int32, device="cuda"), q, kv, torch.randn(260, 64, device="cuda", generator=gen).half(), *cu))

    def run(c):
        ql, qr, table, n, q, kv, kr, cq, ck = c
        return (*K.latent_decode(ql, qr, cache, table, n, 0.07), *K.latent_prefill(q[..., :128], q[..., 128:], kv, kr, cq, ck, 0.07))

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(run(c))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_operators_hold_their_schemas():
    """No hidden writes, and shapes as the fake implementations say; gradients are refused."""
    gen = torch.Generator(device="cuda").manual_seed(4)

    def r(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).half()

    i32, i64 = (lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")), (lambda *v: torch.tensor(v, dtype=torch.int64, device="cuda"))
    cache, ops = r(5, 64, 320), torch.ops.gemq_b200
    decode = (r(2, 1, 4, 256), r(2, 1, 4, 64), cache, i32([0, 1], [2, 3]), i32(100, 7))
    prefill = (r(6, 4, 128), r(6, 4, 64), r(9, 4, 256), r(9, 64), i32(0, 6), i32(0, 9))
    for op, args in ((ops.latent_decode.default, (*decode, 0.1)),
                     (ops.latent_decode_shared.default, (*decode, i32([4, 0]), i32(70), i32(0, 2), 0.1)),
                     (ops.latent_prefill.default, (*prefill, 0.1)),
                     (ops.latent_append.default, (r(3, 320), r(3, 4, 64), r(256), 1e-6, torch.ones(32, device="cuda"), i64(0, 1, 2), i64(5, -1, 64), cache)),
                     (ops.copy_pages.default, (cache, i64(0), i64(4)))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))
    from gemq_b200 import kernels as K
    q = decode[0].requires_grad_()
    with pytest.raises(RuntimeError, match="no autograd formula"):
        K.latent_decode(q, *decode[1:], 0.1)[0].sum().backward()
