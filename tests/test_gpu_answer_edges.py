"""The int8 operators of the text model's answers where calls meet: a text layer and its answer as one run, graphs, streams,
odd addresses, settings at their ends, sizes past 31 bits, refusals."""

import math

import pytest
import torch

from oracle import answer as A
from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops
from tests.test_gpu_answer import BF16, DEV, FP16, FP32, dev, gen, product_inputs, row_inputs, rows_check, tokens_check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    L.device_error(reset=True)
    yield
    torch.cuda.synchronize()
    assert L.device_error(reset=True) == 0


# ----------------------------------------------------------------------------- a layer and its answer

HIDDEN, MLP, HEADS, KV, DIM, VOCAB, PAGE = 320, 608, 5, 1, 64, 1500, 16


def weight(g, n, k, smooth=None):
    w = (torch.randn(n, k, generator=g) / math.sqrt(k)).to(BF16).to(DEV)
    return ops.pack_weight_i8(w, smooth)


class Layer:
    """One layer of a text model and its head, with weights from pack_weight_i8."""

    def __init__(self, seed):
        g = gen(seed)
        self.qkv = weight(g, (HEADS + 2 * KV) * DIM, HIDDEN)
        self.o = weight(g, HIDDEN, HEADS * DIM)
        self.gate_up = weight(g, 2 * MLP, HIDDEN)
        self.smooth = torch.exp(0.4 * torch.randn(MLP, generator=g)).to(DEV)
        self.down = weight(g, HIDDEN, MLP, self.smooth)
        self.head = weight(g, VOCAB, HIDDEN)
        self.norms = [(1 + 0.2 * torch.randn(HIDDEN, generator=g)).to(BF16).to(DEV) for _ in range(3)]
        self.cs = ops.rope_table_wide(256, 10000.0, DEV, DIM)

    def step(self, h, cache, cu, kv_len, table, u, top_p, seen=None):
        """The newest tokens' hidden states -> their next tokens; `seen` collects every stage's inputs and outputs."""
        def note(name, *x):
            if seen is not None:
                seen[name] = x
        r = ops.quantize_rows(h, weight=self.norms[0])
        qkv = ops.linear_i8_rows(r.codes, r.scale, *self.qkv)
        note("in", h, None, self.norms[0], None, r)
        note("qkv", r.codes, r.scale, *self.qkv, None, False, qkv)
        q, k, v = qkv.view(-1, HEADS + 2 * KV, DIM).split([HEADS, KV, KV], 1)
        q = ops.kv_append(cache, k, v, cu, kv_len, table, q=q, rope_cs=self.cs)
        o = ops.paged_attention(q, cache, cu, kv_len, table)
        r = ops.quantize_rows(o.view(-1, HEADS * DIM))
        h2 = ops.linear_i8_rows(r.codes, r.scale, *self.o, residual=h)
        note("attention", o.view(-1, HEADS * DIM), None, None, None, r)
        note("o", r.codes, r.scale, *self.o, h, False, h2)
        r = ops.quantize_rows(h2, weight=self.norms[1])
        m = ops.linear_i8_rows(r.codes, r.scale, *self.gate_up, gated=True)
        note("gated", r.codes, r.scale, *self.gate_up, None, True, m)
        r = ops.quantize_rows(m, smooth=self.smooth)
        d = ops.linear_i8_rows(r.codes, r.scale, *self.down)
        note("smoothed", m, None, None, self.smooth, r)
        note("down", r.codes, r.scale, *self.down, None, False, d)
        r = ops.quantize_rows(d, weight=self.norms[2], residual=h2)
        note("out", d, h2, self.norms[2], None, r)
        logits = ops.linear_i8_rows(r.codes, r.scale, *self.head, dtype=FP32)
        note("logits", r.codes, r.scale, *self.head, None, False, logits)
        return ops.sample_tokens(logits, u, temperature=0.9, top_k=200, top_p=top_p), logits, r.sum


def batch_of(lengths, new, seed):
    """Hidden states of `new` tokens of each sequence behind `lengths` cached ones, and the cache's tables."""
    g = gen(seed)
    pages = [-(-(n + c) // PAGE) for n, c in zip(lengths, new)]
    order, at, table = torch.randperm(sum(pages) + 1, generator=g).tolist(), 0, []
    for p in pages:
        table.append(order[at:at + p] + [0] * (max(pages) - p))
        at += p
    cu = [0] + torch.tensor(new).cumsum(0).tolist()
    cache = torch.randn(sum(pages) + 1, KV, 2, PAGE, DIM, generator=g).to(BF16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return (torch.randn(sum(new), HIDDEN, generator=g).to(BF16).to(DEV), cache.to(DEV), ints(cu),
            ints([n + c for n, c in zip(lengths, new)]), ints(table), torch.rand(sum(new), generator=g).to(DEV))


@pytest.mark.parametrize("new", [[1] * 9, [1, 4, 2, 1, 30, 7]], ids=["single", "several"])
def test_a_layer_and_its_answer(new):
    """Every stage against its plain form on the stage's own inputs, and the tokens against the logits."""
    layer = Layer(1)
    h, cache, cu, kv_len, table, u = batch_of([(13 * i) % 90 for i in range(len(new))], new, 2)
    seen, top_p = {}, torch.full((len(u),), 0.9, device=DEV)
    (tokens, logprob), logits, out = layer.step(h, cache, cu, kv_len, table, u, top_p, seen)
    cpu = lambda t: None if t is None else t.cpu()  # noqa: E731
    for name, v in seen.items():
        if len(v) == 5:
            x, residual, w, smooth, r = v
            rows_check(cpu(x), dict(residual=cpu(residual), weight=cpu(w), bias=None, smooth=cpu(smooth)), r)
        else:
            codes, scale, w, ws, residual, gated, y = v
            ref, size = A.product(cpu(codes), cpu(scale), cpu(w), cpu(ws), None, cpu(residual), gated)
            assert bool(((y.cpu().double() - ref).abs() <= A.product_tolerance(ref, size, y.dtype)).all()), name
    for b in range(len(u)):
        assert int(tokens[b]) == A.sample(logits[b].cpu(), float(u[b]), temperature=0.9, top_k=200, top_p=0.9)[0]
    assert out.shape == h.shape and bool(torch.isfinite(logprob).all())


def test_a_captured_layer_replays_with_new_inputs():
    layer = Layer(3)
    h, cache, cu, kv_len, table, u = batch_of([5, 40, 0, 17], [1] * 4, 4)
    top_p = torch.tensor([0.5, 0.9, 1.0, 0.7], device=DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer.step(h, cache.clone(), cu, kv_len, table, u, top_p)  # warm
    torch.cuda.synchronize()
    graph, cache2 = torch.cuda.CUDAGraph(), cache.clone()
    with torch.cuda.graph(graph, stream=stream):
        (tokens, logprob), logits, out = layer.step(h, cache2, cu, kv_len, table, u, top_p)
    for seed in (5, 6, 7):
        g = gen(seed)
        h.copy_(torch.randn(h.shape, generator=g))
        u.copy_(torch.rand(4, generator=g))
        top_p.copy_(torch.rand(4, generator=g))
        cache2.copy_(cache)
        graph.replay()
        torch.cuda.synchronize()
        (t, p), l, o = layer.step(h, cache.clone(), cu, kv_len, table, u, top_p)
        assert torch.equal(t, tokens) and torch.equal(p, logprob) and torch.equal(l, logits) and torch.equal(o, out)


def test_two_streams_at_once():
    """The same calls on two streams give what one gives: there is no workspace to share."""
    xs = [row_inputs(700, 960, BF16, "rms", seed=s)[0].to(DEV) for s in (1, 2)]
    w = [weight(gen(s), 1600, 960) for s in (3, 4)]
    logits = [torch.randn(40, 49280, generator=gen(s)).to(DEV) for s in (5, 6)]
    u = torch.rand(40, generator=gen(7)).to(DEV)

    def work(i):
        r = ops.quantize_rows(xs[i])
        return (ops.linear_i8_rows(r.codes, r.scale, *w[i]), ops.linear_i8_rows(r.codes[:3], r.scale[:3], *w[i]),
                *ops.sample_tokens(logits[i], u, top_k=300, top_p=0.9))
    alone = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got.append(work(i))
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(alone[i], got[i]))


# ----------------------------------------------------------------------------- results do not depend on the batch

def test_a_row_is_the_same_in_any_batch():
    x, kw = row_inputs(1500, 960, FP16, "layer", residual=True, smooth=True, seed=8)
    kw = {n: dev(t) for n, t in kw.items()}
    whole = ops.quantize_rows(dev(x), **kw)
    w = weight(gen(9), 700, 960)
    y = ops.linear_i8_rows(whole.codes, whole.scale, *w, dtype=FP32)
    for a, b in ((0, 1), (3, 20), (100, 177), (0, 1000)):
        part = ops.quantize_rows(dev(x[a:b]), **{**kw, "residual": kw["residual"][a:b]})
        assert torch.equal(part.codes, whole.codes[a:b]) and torch.equal(part.scale, whole.scale[a:b])
        for impl in (L.LINEAR_FEW, L.LINEAR_MANY):
            assert torch.equal(ops.linear_i8_rows(part.codes, part.scale, *w, dtype=FP32, impl=impl), y[a:b])
    logits = torch.randn(300, 20000, generator=gen(10)).to(DEV)
    u = torch.rand(300, generator=gen(11)).to(DEV)
    all_ = ops.sample_tokens(logits, u, temperature=1.2, top_p=0.95)
    for a, b in ((0, 1), (7, 9), (50, 250)):
        some = ops.sample_tokens(logits[a:b], u[a:b], temperature=1.2, top_p=0.95)
        assert torch.equal(some[0], all_[0][a:b]) and torch.equal(some[1], all_[1][a:b])


# ----------------------------------------------------------------------------- tokens: addresses and settings at their ends

@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_logits_at_odd_addresses(dtype):
    wide = torch.randn(5, 9001, generator=gen(12)).to(dtype).to(DEV)
    for view in (wide[:, 1:], wide[:, 3:9000], wide[:, :8999], wide[1:, 7:2000]):
        tokens_check(view.cpu(), torch.rand(len(view), generator=gen(13)), top_k=40, top_p=0.9)
        got = ops.sample_tokens(view, torch.full((len(view),), 0.4, device=DEV), min_p=0.01)
        want = ops.sample_tokens(view.contiguous(), torch.full((len(view),), 0.4, device=DEV), min_p=0.01)
        assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("vocab", [300, 6000])
def test_settings_at_their_ends(vocab):
    x = (torch.randn(8, vocab, generator=gen(14)) * 3).float()
    u = torch.tensor([0.0, 1.0, 2.0 ** -24, 1 - 2.0 ** -24, 0.5, 0.25, 0.75, 1e-30])
    for t in (1e-38, 1e-20, 1e-9, 1e-7, 1e-4, 1e4, 1e9, 1e30, 3e38):
        tokens_check(x, u, temperature=t)
        tokens_check(x, u, temperature=t, top_k=vocab // 2, top_p=0.9)
        tokens_check(x, u, temperature=t, top_p=0.5, min_p=1e-3)
    for p in (1e-30, 1e-7, 1 - 2.0 ** -24, 1.0, 2.0):
        tokens_check(x, u, top_p=p)
        tokens_check(x, u, top_p=p, top_k=vocab - 1)
    for p in (1e-30, 1e-13, 1e-6, 1 - 2.0 ** -24, 1.0, 1.0000001):
        tokens_check(x, u, min_p=p)
        tokens_check(x, u, min_p=p, top_p=0.99, temperature=5.0)
    # logits far from zero, and huge ones
    tokens_check(x + 1e6, u, top_p=0.8)
    tokens_check(x * 1e30, u, temperature=1e30, top_k=100, top_p=0.8)
    tokens_check(torch.where(x > 0, torch.finfo(FP32).max, torch.finfo(FP32).min), u, top_p=0.5)
    tokens_check(torch.where(x > 0, torch.finfo(FP32).max, torch.finfo(FP32).min), u, temperature=3e38, top_p=0.7)


@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0, 30.0])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_flat_rows_cut_anywhere(dtype, temperature):
    """Distributions in which top_p and top_k keep thousands, negative and positive logits on both sides of the cut."""
    x = torch.randn(8, 30000, generator=gen(15)).to(dtype)
    x[4:] *= 0.01
    u = torch.rand(8, generator=gen(16))
    tokens_check(x, u, temperature=temperature, top_p=[0.05, 0.3, 0.5, 0.77, 0.9, 0.97, 0.999, 0.6])
    tokens_check(x, u, temperature=temperature, top_k=[257, 1000, 5000, 12345, 20000, 29999, 300, 15000])
    tokens_check(x, u, temperature=temperature, top_p=0.8, min_p=0.02, top_k=[400, 1000, 5000, 12345, 20000, 29999, 300, 15000])


# ----------------------------------------------------------------------------- sizes past 31 bits

def test_rows_beyond_31_bits():
    m, k = 70000, 32768  # 2.3e9 elements
    x = torch.empty(m, k, dtype=BF16, device=DEV)
    x.copy_(torch.linspace(-1, 1, k, device=DEV).to(BF16).expand(m, k))
    x[-1] *= 3
    got = ops.quantize_rows(x)
    want = ops.quantize_rows(x[-2:].clone())
    assert torch.equal(got.codes[-2:], want.codes) and torch.equal(got.scale[-2:], want.scale)
    del got
    # outputs of as many: every row of the product is one row's
    g = gen(17)
    w, ws = torch.randint(-127, 128, (k, 16), generator=g, dtype=torch.int8).to(DEV), torch.rand(k, generator=g).to(DEV)
    rows = torch.randint(-127, 128, (m, 16), generator=g, dtype=torch.int8).to(DEV)
    scale = torch.rand(m, generator=g).to(DEV)
    y = ops.linear_i8_rows(rows, scale, w, ws, out=x)
    assert torch.equal(y[-3:], ops.linear_i8_rows(rows[-3:], scale[-3:], w, ws))
    assert torch.equal(y[65530:65540], ops.linear_i8_rows(rows[65530:65540], scale[65530:65540], w, ws))
    logits = y[:, :k]
    t, _ = ops.sample_tokens(logits, torch.full((m,), 0.5, device=DEV), temperature=0.0)
    assert torch.equal(t[-4:].long(), logits[-4:].float().argmax(-1))


# ----------------------------------------------------------------------------- custom ops and refusals

def test_custom_ops():
    x, kw = row_inputs(20, 77, BF16, "rms", residual=True, seed=18)
    kw = {n: dev(t) for n, t in kw.items()}
    codes, scale, total = torch.ops.svla.quantize_rows(dev(x), kw["weight"], None, 1e-5, kw["residual"], None)
    r = ops.quantize_rows(dev(x), weight=kw["weight"], residual=kw["residual"])
    assert torch.equal(codes, r.codes) and torch.equal(scale, r.scale) and torch.equal(total, r.sum)
    cx, cs, cw, cws = (dev(t) for t in product_inputs(20, 32, 64))
    y = torch.ops.svla.linear_i8_rows(cx, cs, cw, cws, None, None, False, FP16)
    assert torch.equal(y, ops.linear_i8_rows(cx, cs, cw, cws, dtype=FP16))
    u = torch.rand(20, generator=gen(19)).to(DEV)
    t, p = torch.ops.svla.sample_tokens(y, u, None, None, None, None)
    assert torch.equal(t, ops.sample_tokens(y, u)[0]) and torch.equal(p, ops.sample_tokens(y, u)[1])
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fake = [mode.from_tensor(t) for t in (dev(x), kw["weight"], kw["residual"])]
        c, s, total = torch.ops.svla.quantize_rows(fake[0], fake[1], None, 1e-5, fake[2], None)
        assert c.shape == (20, 77) and c.stride() == codes.stride() and s.shape == (20,) and total.shape == (20, 77)


def test_refusals_of_tensors():
    x = torch.zeros(4, 64, dtype=BF16, device=DEV)
    q = torch.zeros(4, 64, dtype=torch.int8, device=DEV)
    s4, s8 = torch.ones(4, device=DEV), torch.ones(8, device=DEV)
    w8 = torch.zeros(8, 64, dtype=torch.int8, device=DEV)
    cases = [
        (lambda: ops.quantize_rows(x.float()), "bf16 or fp16"),
        (lambda: ops.quantize_rows(x[0]), "bf16 or fp16"),
        (lambda: ops.quantize_rows(x.t()), "contiguous rows"),
        (lambda: ops.quantize_rows(x[:1].expand(4, 64)), "overlapping"),
        (lambda: ops.quantize_rows(x, weight=s4), "weight must be"),
        (lambda: ops.quantize_rows(x, weight=torch.ones(64, dtype=FP16, device=DEV)), "weight must be"),
        (lambda: ops.quantize_rows(x, residual=x[:2]), "residual must be"),
        (lambda: ops.quantize_rows(x, smooth=torch.ones(64)), "smooth must be"),
        (lambda: ops.quantize_rows(x, codes=torch.zeros(4, 64, device=DEV)), "codes must be"),
        (lambda: ops.quantize_rows(x, scale=s8), "scale must be"),
        (lambda: ops.linear_i8_rows(x, s4, w8, s8), "x must be"),
        (lambda: ops.linear_i8_rows(q, s8, w8, s8), "x_scale must be"),
        (lambda: ops.linear_i8_rows(q, s4, w8[:, :32], s8), "weight must be"),
        (lambda: ops.linear_i8_rows(q, s4, w8, s4), "wscale must be"),
        (lambda: ops.linear_i8_rows(q, s4, w8[:7], s8[:7], gated=True), "gate and up"),
        (lambda: ops.linear_i8_rows(q, s4, w8, s8, dtype=torch.int32), "dtype"),
        (lambda: ops.linear_i8_rows(q, s4, w8, s8, bias=s4), "bias must be"),
        (lambda: ops.linear_i8_rows(q, s4, w8, s8, residual=torch.zeros(4, 8, device=DEV)), "residual must be"),
        (lambda: ops.linear_i8_rows(q, s4, w8, s8, out=torch.zeros(4, 9, device=DEV)), "out must be"),
        (lambda: ops.sample_tokens(q, s4), "logits must be"),
        (lambda: ops.sample_tokens(x, s8), "u must be"),
        (lambda: ops.sample_tokens(x, s4, temperature=s8), "temperature must be"),
        (lambda: ops.sample_tokens(x, s4, top_k=torch.ones(4, dtype=torch.int64, device=DEV)), "top_k must be"),
        (lambda: ops.sample_tokens(x, s4, tokens=s4), "tokens must be"),
    ]
    for call, word in cases:
        with pytest.raises(ValueError, match=word):
            call()
    library = [
        (lambda: ops.linear_i8_rows(q[:, :60].contiguous(), s4, w8[:, :60], s8), "16"),
        (lambda: ops.linear_i8_rows(q[:, 8:40], s4, w8[:, :32], s8), "16-byte"),
        (lambda: ops.linear_i8_rows(q, s4, w8, s8, gated=True, bias=torch.zeros(4, device=DEV)), "gated"),
        (lambda: ops.quantize_rows(x, bias=x[0]), "bias without weight"),
        (lambda: ops.quantize_rows(x, eps=-1.0), "eps"),
        (lambda: ops.sample_tokens(x, s4, temperature=-1.0), "temperature"),
        (lambda: ops.sample_tokens(x, s4, top_p=math.nan), "top_p"),
    ]
    for call, word in library:
        with pytest.raises(L.SvlaError, match=word):
            call()


def test_empty_calls():
    x = torch.zeros(0, 64, dtype=BF16, device=DEV)
    r = ops.quantize_rows(x, residual=x, want_values=True)
    assert r.codes.shape == (0, 64) and r.scale.shape == (0,) and r.sum.shape == (0, 64)
    w, ws = torch.zeros(8, 64, dtype=torch.int8, device=DEV), torch.ones(8, device=DEV)
    assert ops.linear_i8_rows(r.codes, r.scale, w, ws).shape == (0, 8)
    q = torch.zeros(3, 64, dtype=torch.int8, device=DEV)
    assert ops.linear_i8_rows(q, torch.ones(3, device=DEV), w[:0], ws[:0]).shape == (3, 0)
    t, p = ops.sample_tokens(torch.zeros(0, 5, device=DEV), torch.zeros(0, device=DEV))
    assert t.shape == (0,) and p.shape == (0,)


def test_what_is_not_finite_stays_visible():
    """A row with an infinity gives NaN in every product, and its logits no token."""
    x, _ = row_inputs(4, 960, BF16, seed=20)
    x[2, 17] = math.inf
    r = ops.quantize_rows(dev(x), weight=torch.ones(960, dtype=BF16, device=DEV))
    w = weight(gen(21), 300, 960)
    for impl in (L.LINEAR_FEW, L.LINEAR_MANY):
        y = ops.linear_i8_rows(r.codes, r.scale, *w, dtype=FP32, impl=impl)
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isfinite(y[[0, 1, 3]]).all())
        g = ops.linear_i8_rows(r.codes, r.scale, *w, gated=True, dtype=FP32, impl=impl)
        assert bool(torch.isnan(g[2]).all()) and bool(torch.isfinite(g[[0, 1, 3]]).all())
    t, p = ops.sample_tokens(y, torch.full((4,), 0.5, device=DEV), top_k=10)
    assert int(t[2]) == -1 and math.isnan(float(p[2])) and bool((t[[0, 1, 3]] >= 0).all())
