"""The serving operators on the GPU against plain forms in 64 bits (oracle/serving.py).

Bars.  Attention: the bound that oracle.serving.attention_tolerance derives from the roundings the kernels make.
Appending: bit-exact with the same fp32 operations done one by one on the CPU -- cache bytes, rotated rows, rows as held --
and every other byte of the cache left as it was.
"""

import math

import pytest
import torch

from oracle import serving as S
from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_device_error():
    L.device_error(reset=True)
    yield
    torch.cuda.synchronize()
    assert L.device_error(reset=True) == 0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def starts(lens):
    return [0] + torch.tensor(lens).cumsum(0).tolist()


def within(got, ref, tol, what=""):
    got, bad = got.double().cpu(), None
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    ok = ((got - ref).abs() <= tol) | (got == ref) | torch.isnan(ref)
    if not bool(ok.all()):
        bad = ((got - ref).abs() / tol)[~ok].max()
    assert bool(ok.all()), (what, int((~ok).sum()), float(bad))


# ----------------------------------------------------------------------------- packed prompts

def packed_inputs(lens_q, lens_k, hq, hkv, d, dtype, seed=0, q_scale=1.0, extra=0):
    """q [sum + extra, hq, d]; k and v are parts of one [sum + extra, 2 hkv, d] buffer, as a projection leaves them."""
    g = gen(seed)
    q = (torch.randn(sum(lens_q) + extra, hq, d, generator=g) * q_scale).to(dtype)
    kv = torch.randn(sum(lens_k) + extra, 2 * hkv, d, generator=g).to(dtype)
    return q, kv


def packed_reference(q, kv, lens_q, lens_k, causal, scale=None):
    hkv, d = kv.shape[1] // 2, q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    aq, ak, outs = starts(lens_q), starts(lens_k), []
    for b in range(len(lens_q)):
        k, v = kv[ak[b]:ak[b + 1], :hkv].double(), kv[ak[b]:ak[b + 1], hkv:].double()
        outs.append(S.attend_dense(q[aq[b]:aq[b + 1]].double(), k, v, S.causal_seen(lens_q[b], lens_k[b], causal), scale)
                    if lens_q[b] and lens_k[b] else
                    [torch.zeros(lens_q[b], q.shape[1], d, dtype=torch.float64)] * 2 +
                    [torch.zeros(lens_q[b], q.shape[1], dtype=torch.float64)])
    return [torch.cat([o[i] for o in outs]) for i in range(3)]


KERNELS = [L.ATTN_MMA_SYNC, L.ATTN_TCGEN05]


def packed_check(lens_q, lens_k, hq, hkv, d, dtype, causal=True, seed=0, q_scale=1.0):
    q, kv = packed_inputs(lens_q, lens_k, hq, hkv, d, dtype, seed, q_scale)
    o, spread, size = packed_reference(q, kv, lens_q, lens_k, causal)
    kvd = kv.to(DEV)
    for impl in KERNELS:
        got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints(starts(lens_q)).to(DEV),
                                   ints(starts(lens_k)).to(DEV), causal=causal, impl=impl)
        within(got, o, S.attention_tolerance(o, spread, size, dtype, d), f"impl {impl}")


LENGTHS = [
    ([1], [1]), ([2], [2]), ([177], [177]), ([1, 2, 3, 1], [1, 2, 3, 1]),
    ([63, 64, 65, 128, 129, 1], [63, 64, 65, 128, 129, 1]),
    ([5, 1, 17], [80, 300, 17]),        # the last tokens of longer sequences
    ([9, 4, 3], [4, 0, 3]),             # fewer keys than queries, none at all
    ([0, 7, 0, 0, 3, 0], [0, 7, 5, 0, 3, 0]),
    ([300, 41], [300, 700]),
]


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(15, 5, 64), (4, 4, 64), (8, 2, 128), (7, 1, 128)], ids=str)
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_packed_attention(lens, heads, dtype):
    packed_check(*lens, *heads, dtype)


@pytest.mark.parametrize("heads", [(15, 5, 64), (3, 1, 128), (64, 1, 64), (33, 1, 128), (20, 1, 64)], ids=str)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_head_groups_and_both_directions(heads, causal):
    packed_check([130, 1, 45, 260], [130, 64, 200, 260], *heads, BF16, causal=causal, seed=3)


@pytest.mark.parametrize("heads", [(15, 5, 64), (8, 2, 128)], ids=str)
def test_packed_attention_long_and_many(heads):
    packed_check([1500], [1500], *heads, BF16, seed=4)
    lens = [1 + (7 * i) % 23 for i in range(150)]
    packed_check(lens, lens, *heads, FP16, seed=5)


@pytest.mark.parametrize("n", [127, 128, 129, 1000])
def test_packed_attention_finds_every_tile_of_many_sequences(n):
    """Lengths of nothing, of less than a tile, of whole tiles (21 and 42 tokens at 3 heads) and of several."""
    lens = [(0, 1, 21, 42, 43, 7, 130)[(i * i + i // 9) % 7] for i in range(n)]
    packed_check(lens, lens, 3, 1, 64, BF16, seed=33)


@pytest.mark.parametrize("impl", KERNELS)
def test_packed_attention_with_sharp_and_growing_scores(impl):
    """Scores over a range of hundreds, and keys that grow along the sequence, so that the running maximum moves all the
    time."""
    for d, hq, hkv in ((64, 3, 1), (128, 4, 2)):
        packed_check([400], [400], hq, hkv, d, BF16, seed=6, q_scale=12.0)
        q, kv = packed_inputs([500], [500], hq, hkv, d, BF16, seed=7)
        ramp = torch.linspace(0.05, 6.0, 500)[:, None, None]
        kv[:, :hkv] = (q[:, :1].float().mean(0, keepdim=True) * 0 + q[0, :1].float() * ramp).to(BF16)
        q = q[:1].expand(500, hq, d).contiguous()
        o, spread, size = packed_reference(q, kv, [500], [500], True)
        kvd = kv.to(DEV)
        got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints([0, 500]).to(DEV), impl=impl)
        within(got, o, S.attention_tolerance(o, spread, size, BF16, d))


@pytest.mark.parametrize("impl", KERNELS)
def test_packed_attention_scale_and_strided_rows(impl):
    lens, hq, hkv, d = [70, 3], 6, 2, 64
    q, kv = packed_inputs(lens, lens, hq, hkv, d, BF16, seed=8)
    o, spread, size = packed_reference(q, kv, lens, lens, True, scale=0.3)
    fused = torch.cat([q, kv, torch.full((73, 1, d), float("nan"), dtype=BF16)], 1).to(DEV)  # rows of 11 heads
    out = torch.full((73, 9, d), 7.0, dtype=BF16, device=DEV)
    cu = ints(starts(lens)).to(DEV)
    got = ops.packed_attention(fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:hq + 2 * hkv], cu, scale=0.3,
                               out=out[:, 2:8], impl=impl)
    within(got, o, S.attention_tolerance(o, spread, size, BF16, d))
    assert bool((out[:, :2] == 7).all()) and bool((out[:, 8:] == 7).all())


@pytest.mark.parametrize("heads", [(15, 5, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("impl", KERNELS)
def test_packed_attention_keeps_sequences_apart(impl, heads, dtype, fill):
    """A sequence full of NaN or infinities between two others, and rows behind the last one: the others' results are
    those without them, and rows behind the last sequence are left as they were."""
    hq, hkv, d = heads
    lens = [50, 30, 131]
    q, kv = packed_inputs(lens, lens, hq, hkv, d, dtype, seed=9, extra=60)
    o, spread, size = packed_reference(q, kv, lens, lens, True)
    q[50:80], kv[50:80] = fill, fill
    q[211:], kv[211:] = fill, fill
    out = torch.full_like(q, 3.0).to(DEV)
    kvd = kv.to(DEV)
    ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints(starts(lens)).to(DEV), out=out, impl=impl)
    tol = S.attention_tolerance(o, spread, size, dtype, d)
    for a, b in ((0, 50), (80, 211)):
        within(out[a:b], o[a:b], tol[a:b])
    assert bool((out[211:] == 3).all())


@pytest.mark.parametrize("heads", [(15, 5, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("n,at", [(40, 20), (200, 130), (200, 0), (300, 299), (300, 127), (300, 128)])
@pytest.mark.parametrize("impl", KERNELS)
def test_packed_attention_non_finite_value_reaches_only_the_rows_that_see_it(impl, heads, n, at):
    hq, hkv, d = heads
    q, kv = packed_inputs([n], [n], hq, hkv, d, BF16, seed=10)
    o, spread, size = packed_reference(q, kv, [n], [n], True)
    kv[at, hkv, 3], kv[at, hkv, 5], kv[at, hkv + 1, d - 1] = float("nan"), float("inf"), -float("inf")
    g = hq // hkv
    o[at:, :g, 3], o[at:, :g, 5], o[at:, g:2 * g, d - 1] = float("nan"), float("inf"), -float("inf")
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints([0, n]).to(DEV), impl=impl)
    within(got, o, S.attention_tolerance(o, spread, size, BF16, d).nan_to_num(1.0))


@pytest.mark.parametrize("impl", KERNELS)
def test_packed_attention_non_finite_queries_and_keys(impl):
    """A NaN in a query row spoils that row alone; one in a key, the rows that see it."""
    hq, hkv, d, n = 6, 2, 64, 150
    q, kv = packed_inputs([n], [n], hq, hkv, d, BF16, seed=11)
    o, spread, size = packed_reference(q, kv, [n], [n], True)
    q[10, 1, 0] = float("nan")
    kv[100, 1, 7] = float("nan")
    o[10, 1] = float("nan")
    o[100:, 3:] = float("nan")
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints([0, n]).to(DEV), impl=impl)
    within(got, o, S.attention_tolerance(o, spread, size, BF16, d))


@pytest.mark.parametrize("impl", KERNELS)
@pytest.mark.parametrize("heads", [(3, 1, 64), (4, 2, 128)], ids=str)
def test_packed_attention_nan_score_at_any_place_spoils_its_rows(impl, heads):
    """One sequence per place of the NaN key: whichever way its exponential is computed, the rows that see it are NaN."""
    hq, hkv, d, n = *heads, 145
    places = list(range(0, 20)) + [32, 33, 63, 64, 80, 113, 127, 128, 129, 144]
    lens = [n] * len(places)
    q, kv = packed_inputs(lens, lens, hq, hkv, d, BF16, seed=34)
    for i, j in enumerate(places):
        kv[i * n + j, :hkv, 3] = float("nan")
    cu = ints(starts(lens)).to(DEV)
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], cu, impl=impl).isnan().flatten(1).cpu()
    for i, j in enumerate(places):
        rows = got[i * n:(i + 1) * n]
        assert not rows[:j].any() and rows[j:].all(), f"place {j}"


@pytest.mark.parametrize("impl", KERNELS)
def test_packed_attention_bounds_its_rows_by_the_tensors(impl):
    """Starts that point behind the tensors are cut off there; nothing outside is read or written."""
    q, kv = packed_inputs([20], [20], 6, 2, 64, BF16, seed=12)
    kvd = kv.to(DEV)
    ref = ops.packed_attention(q.to(DEV), kvd[:, :2], kvd[:, 2:], ints([0, 20]).to(DEV), impl=impl)
    got = ops.packed_attention(q.to(DEV), kvd[:, :2], kvd[:, 2:], ints([0, 1 << 20]).to(DEV), impl=impl)
    assert torch.equal(got, ref)
    none = ops.packed_attention(q.to(DEV), kvd[:0, :2], kvd[:0, 2:], ints([0, 20]).to(DEV), ints([0, 0]).to(DEV))
    assert bool((none == 0).all())
    if impl == L.ATTN_TCGEN05:
        with pytest.raises(L.SvlaError, match="needs keys"):
            ops.packed_attention(q.to(DEV), kvd[:0, :2], kvd[:0, 2:], ints([0, 20]).to(DEV), ints([0, 0]).to(DEV), impl=impl)


@pytest.mark.parametrize("impl", KERNELS)
def test_packed_attention_repeats_replays_and_other_streams(impl):
    lens = [33, 190, 1]
    q, kv = packed_inputs(lens, lens, 15, 5, 64, BF16, seed=13)
    q, kv, cu = q.to(DEV), kv.to(DEV), ints(starts(lens)).to(DEV)
    call = lambda: ops.packed_attention(q, kv[:, :5], kv[:, 5:], cu, impl=impl)  # noqa: E731
    ref = call()
    assert all(torch.equal(call(), ref) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    q2, _ = packed_inputs(lens, lens, 15, 5, 64, BF16, seed=14)
    q.copy_(q2)
    cu.copy_(ints(starts([100, 120, 4])))  # the lengths are the device's: a replay follows them
    graph.replay()
    replayed = held.clone()
    assert torch.equal(replayed, call())


# ----------------------------------------------------------------------------- appending

def make_table(lens, page, seed=0, spare=2, width=None):
    """(page_table [B, width], number of pages): every sequence's pages in random order; unused columns are -1."""
    need = [max(1, -(-n // page)) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=gen(seed)).tolist()
    table = torch.full((len(lens), max(need) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ints(order[at:at + n])
        at += n
    return table, sum(need) + spare


def random_cache(n_pages, page, hkv, d, bits, dtype, seed=0):
    """Whatever bytes were there before: for 16 bits normal numbers, for 4 bits random bytes."""
    c = ops.kv_cache(n_pages, page, hkv, d, bits, dtype, device="cpu")
    if bits == 16:
        return torch.randn(c.shape, generator=gen(seed)).to(dtype)
    return torch.randint(0, 256, c.shape, generator=gen(seed), dtype=torch.uint8)


def append_case(new, past, heads, dtype, bits, page, seed=0, with_q=True, pos=None, rope=True, extra=0):
    hq, hkv, d = heads
    g = gen(seed)
    T = sum(new) + extra
    q, k, v = (torch.randn(T, h, d, generator=g).to(dtype) for h in (hq, hkv, hkv))
    total = [a + b for a, b in zip(new, past)]
    table, n_pages = make_table(total, page, seed)
    cache = random_cache(n_pages, page, hkv, d, bits, dtype, seed)
    cs = ops.rope_table_wide(max(total) + 5, 10000.0, DEV, d) if rope else None
    dev = {n: (None if t is None else t.to(DEV)) for n, t in dict(
        cache=cache, k=k, v=v, cu_q=ints(starts(new)), kv_len=ints(total), table=table, q=q if with_q else None,
        pos=None if pos is None else ints(pos)).items()}
    want = cache.clone()
    rq, rk, rv = S.append(want, page, k, v, starts(new), total, table, None if cs is None else cs.cpu(), pos,
                          q if with_q else None)
    gq, gk, gv = ops.kv_append(dev["cache"], dev["k"], dev["v"], dev["cu_q"], dev["kv_len"], dev["table"], q=dev["q"],
                               rope_cs=cs, pos=dev["pos"], want_rows=True)
    n = sum(new)
    assert torch.equal(dev["cache"].cpu().view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(gk[:n].cpu(), rk[:n]) and torch.equal(gv[:n].cpu(), rv[:n])
    if with_q:
        assert torch.equal(gq[:n].cpu(), rq[:n])
    else:
        assert gq is None


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads", [(15, 5, 64), (8, 1, 128), (32, 8, 128), (12, 12, 64)], ids=str)
@pytest.mark.parametrize("new,past,page", [([1], [0], 16), ([1], [177], 16), ([1, 1, 1, 1, 1], [15, 16, 17, 0, 63], 16),
                                           ([70, 0, 1, 33], [0, 9, 100, 31], 48), ([200], [3], 256)])
def test_kv_append_is_exact(new, past, page, heads, bits, dtype):
    append_case(new, past, heads, dtype, bits, page)


@pytest.mark.parametrize("bits", [16, 4])
def test_kv_append_many_sequences(bits):
    new = [(i * 5) % 4 for i in range(1100)]
    append_case(new, [i % 37 for i in range(1100)], (2, 2, 64), BF16, bits, 16, seed=2)
    append_case([1] * 200, [i for i in range(200)], (15, 5, 64), BF16, bits, 32, seed=3)


@pytest.mark.parametrize("bits", [16, 4])
def test_kv_append_without_queries_rotation_or_with_positions(bits):
    append_case([3, 4], [10, 20], (4, 2, 64), BF16, bits, 16, with_q=False)
    append_case([3, 4], [10, 20], (4, 2, 64), BF16, bits, 16, rope=False)
    append_case([3, 4], [10, 20], (4, 2, 128), FP16, bits, 16, pos=[0, 1, 2, 5, 0, 24, 7])
    append_case([3], [10], (4, 2, 64), BF16, bits, 16, pos=[-1, 3, 100000])  # clamped to the table
    append_case([3, 4], [10, 20], (4, 2, 64), BF16, bits, 16, extra=9)       # rows behind the last sequence


@pytest.mark.parametrize("bits", [16, 4])
def test_kv_append_in_place_and_strided(bits):
    hq, hkv, d, new = 6, 2, 64, [5, 2]
    x = torch.randn(9, hq + 2 * hkv, d, generator=gen(4)).to(BF16)
    q, k, v = x.split([hq, hkv, hkv], 1)
    table, n_pages = make_table([5, 2], 16)
    cache = ops.kv_cache(n_pages, 16, hkv, d, bits, device=DEV)
    want = cache.cpu().clone()
    cs = ops.rope_table_wide(16, 10000.0, DEV, d)
    rq, rk, rv = S.append(want, 16, k, v, [0, 5, 7], [5, 2], table, cs.cpu(), None, q)
    xd = x.to(DEV)
    qd, kd, vd = xd.split([hq, hkv, hkv], 1)
    ops.kv_append(cache, kd, vd, ints([0, 5, 7]).to(DEV), ints([5, 2]).to(DEV), table.to(DEV), q=qd, rope_cs=cs,
                  q_out=qd, k_out=kd, v_out=vd)
    assert torch.equal(xd[:7].cpu(), torch.cat([rq, rk, rv], 1)[:7])
    assert torch.equal(xd[7:].cpu(), x[7:])  # rows behind the last sequence stay as they were
    assert torch.equal(cache.cpu().view(torch.uint8), want.view(torch.uint8))


def test_kv_append_extreme_groups():
    """Groups of one value, of zeros, of the type's largest values, and with NaN or infinities (they read back as NaN)."""
    d, page = 64, 16
    k = torch.randn(6, 1, d, generator=gen(5)).to(BF16)
    v = k.clone()
    k[0], v[0] = 0.0, 2.5
    k[1, 0, :32] = torch.finfo(BF16).max / 4
    k[2, 0, 40], v[2, 0, 3] = float("nan"), float("inf")
    v[3, 0, :] = 1e-30
    v[4, 0, 5] = 1e4
    table, n_pages = make_table([6], page)
    cache = ops.kv_cache(n_pages, page, 1, d, 4, device=DEV)
    _, gk, gv = ops.kv_append(cache, k.to(DEV), v.to(DEV), ints([0, 6]).to(DEV), ints([6]).to(DEV), table.to(DEV),
                              want_rows=True)
    want = cache.cpu().clone()
    _, rk, rv = S.append(want, page, k, v, [0, 6], [6], table)
    for got, ref in ((gk, rk), (gv, rv)):
        got = got.cpu()
        nan = torch.isnan(ref)
        assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], ref[~nan])
    assert bool(torch.isnan(gk[2, 0, 32:]).all()) and bool(torch.isfinite(gk[2, 0, :32]).all())
    assert bool(torch.isnan(gv[2, 0, :32]).all()) and bool(torch.isfinite(gv[2, 0, 32:]).all())


@pytest.mark.parametrize("bits", [16, 4])
def test_kv_append_skips_entries_outside_the_cache(bits):
    """A page outside the cache, an entry outside the table: those rows are left out, the others are written, and the
    device error word says so."""
    new, total, page = [2, 2, 2], [18, 5, 60], 16
    k = torch.randn(6, 2, 64, generator=gen(6)).to(BF16)
    table = ints([[0, 7], [1, 0], [2, 3]])  # sequence 0's second page does not exist; sequence 2 needs a fourth column
    cache = ops.kv_cache(4, page, 2, 64, bits, device=DEV)
    want = cache.cpu().clone()
    S.append(want, page, k, k, starts(new), total, table)
    ops.kv_append(cache, k.to(DEV), k.to(DEV), ints(starts(new)).to(DEV), ints(total).to(DEV), table.to(DEV))
    assert torch.equal(cache.cpu().view(torch.uint8), want.view(torch.uint8))
    assert L.device_error(reset=True) == L.ERR_BAD_PAGE


def test_rope_table_wide_keeps_far_angles():
    """(cos, sin) rounded to fp32 from 64-bit angles: half a step of fp32 at 1 (2^-25), and the 64-bit angle's own error
    (position 2^17 times 2^-52)."""
    n, d = 131072, 128
    cs = ops.rope_table_wide(n, 10000.0, DEV, d).cpu().double()
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(d // 2, dtype=torch.float64) / (d // 2))
    ref = torch.stack([angle.cos(), angle.sin()], -1)
    assert float((cs - ref).abs().max()) <= 2.0 ** -25 + 2.0 ** -33


# ----------------------------------------------------------------------------- paged attention

def filled_cache(lens, heads, bits, page, dtype, seed=0, rest=float("nan"), width=None):
    """A cache holding random entries of the sequences; every other entry is `rest` (NaN: nobody may look at it)."""
    _, hkv, d = heads
    table, n_pages = make_table(lens, page, seed, width=width)
    cache = ops.kv_cache(n_pages, page, hkv, d, bits, dtype, device="cpu")
    if bits == 16:
        cache.fill_(rest)
    else:
        cache.fill_(255)  # codes 15, (step, low) = NaN
    g = gen(seed)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k, v = torch.randn(n, hkv, d, generator=g), torch.randn(n, hkv, d, generator=g)
        k[..., 5] *= 4
        S.append(cache, page, k.to(dtype), v.to(dtype), [0, n], [n], table[b:b + 1])
    return cache, table


def paged_reference(q, cache, page, table, new, total, scale=None):
    d, at, outs = q.shape[2], starts(new), []
    scale = d ** -0.5 if scale is None else scale
    for b in range(len(new)):
        k, v, ks, vs = S.rows(cache, page, d, table[b], total[b])
        outs.append(S.attend_dense(q[at[b]:at[b + 1]].double(), k, v, S.causal_seen(new[b], total[b]), scale, ks, vs)
                    if total[b] and new[b] else
                    [torch.zeros(new[b], q.shape[1], d, dtype=torch.float64)] * 2 +
                    [torch.zeros(new[b], q.shape[1], dtype=torch.float64)])
    return [torch.cat([o[i] for o in outs]) for i in range(3)]


def paged_tolerance(o, spread, size, dtype, d, bits, total, top):
    """4 bits: the weights p step are rounded to fp16 (half a step 2^-11 relative); weights below 2^-14 of the largest
    are subnormal, off by 2^-25 of at most twice the largest step, for each of the entries, times a code of 15."""
    if bits == 16:
        return S.attention_tolerance(o, spread, size, dtype, d)
    return S.attention_tolerance(o, spread, size, dtype, d, weight_unit=2.0 ** -11,
                                 floor=max(total) * 15 * 2.0 ** -25 * 2 * top)


def paged_check(new, past, heads, bits, page, dtype, seed=0, q_scale=1.0, width=None, scale=0.0):
    hq, hkv, d = heads
    total = [a + b for a, b in zip(new, past)]
    cache, table = filled_cache(total, heads, bits, page, dtype, seed, width=width)
    q = (torch.randn(sum(new), hq, d, generator=gen(seed + 100)) * q_scale).to(dtype)
    o, spread, size = paged_reference(q, cache, page, table, new, total, scale or None)
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints(starts(new)).to(DEV), ints(total).to(DEV), table.to(DEV),
                              scale=scale)
    within(got, o, paged_tolerance(o, spread, size, dtype, d, bits, total, top=1.0))  # steps of 8 sigma / 15 stay below 1
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads", [(15, 5, 64), (8, 1, 128), (4, 4, 64), (6, 2, 128)], ids=str)
@pytest.mark.parametrize("new,past,page", [
    ([1], [0], 16), ([1], [177], 16), ([1, 1, 1, 1, 1, 1], [14, 15, 16, 31, 32, 64], 16),
    ([1, 1], [700, 3], 64), ([3, 5, 2], [0, 40, 100], 48)])
def test_paged_attention(new, past, page, heads, bits, dtype):
    paged_check(new, past, heads, bits, page, dtype)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads", [(15, 5, 64), (32, 8, 128)], ids=str)
def test_paged_attention_split_over_the_gpu(heads, bits):
    """Long and short sequences: pieces cut the long ones, and several short ones share a piece."""
    paged_check([1, 1, 1, 1], [4999, 2, 1234, 0], heads, bits, 16, BF16, seed=21)
    paged_check([2, 1], [6000, 300], heads, bits, 32, FP16, seed=22)
    paged_check([1] * 40, [(i * 131) % 900 for i in range(40)], heads, bits, 16, BF16, seed=23)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads,new", [((3, 1, 64), 1), ((8, 1, 128), 1), ((5, 1, 128), 3), ((4, 1, 64), 2)], ids=str)
def test_paged_attention_joins_many_parts(heads, new, bits):
    """One kv head: all pieces belong to one item, whose parts' maxima lie far apart."""
    paged_check([new], [13000], heads, bits, 64, BF16, seed=30, q_scale=4.0)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads", [(3, 1, 64), (16, 1, 64), (9, 1, 128), (71, 1, 64), (40, 2, 128)], ids=str)
def test_paged_attention_head_groups_and_drafts(heads, bits):
    paged_check([1, 1], [100, 33], heads, bits, 16, BF16, seed=24)
    paged_check([7, 1, 0, 20], [100, 33, 12, 5], heads, bits, 16, BF16, seed=25)
    paged_check([130], [20], heads, bits, 16, FP16, seed=26)


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_attention_sharp_scores_scale_and_wide_tables(bits):
    paged_check([1, 2], [300, 500], (6, 2, 64), bits, 16, BF16, seed=27, q_scale=12.0)
    paged_check([1, 2], [300, 500], (6, 2, 128), bits, 16, FP16, seed=28, scale=0.25)
    paged_check([1, 2], [3, 50], (6, 2, 64), bits, 16, BF16, seed=29, width=400)  # room for more than there is


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_attention_sequences_without_entries_or_tokens(bits):
    hq, hkv, d = 6, 2, 64
    new, total = [1, 0, 3, 2], [0, 20, 2, 40]  # sequence 2: more tokens than entries, its first row sees nothing
    cache, table = filled_cache(total, (hq, hkv, d), bits, 16, BF16)
    q = torch.randn(sum(new) + 4, hq, d, generator=gen(1)).to(BF16)
    o, spread, size = paged_reference(q[:6], cache, 16, table, new, total)
    out = torch.full_like(q, 9.0).to(DEV)
    ops.paged_attention(q.to(DEV), cache.to(DEV), ints(starts(new)).to(DEV), ints(total).to(DEV), table.to(DEV), out=out)
    within(out[:6], o, paged_tolerance(o, spread, size, BF16, d, bits, total, 1.0))
    assert bool((out[0] == 0).all()) and bool((out[1] == 0).all())
    assert bool((out[6:] == 9).all())  # rows behind the last sequence stay as they were


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("width", [None, 64], ids=["one piece", "pieces"])
def test_paged_attention_non_finite_values_reach_only_the_rows_that_see_them(bits, width):
    hq, hkv, d, new, total = 6, 2, 64, [5], [45]
    cache, table = filled_cache(total, (hq, hkv, d), bits, 16, BF16, seed=3, width=width)
    q = torch.randn(5, hq, d, generator=gen(2)).to(BF16)
    o, spread, size = paged_reference(q, cache, 16, table, new, total)
    pid, slot = int(table[0, 42 // 16]), 42 % 16  # entry 42: rows 2, 3 and 4 see it
    if bits == 16:
        cache[pid, 0, 1, slot, 7] = float("nan")
        o[2:, :3, 7] = float("nan")
    else:
        S.split4(cache[pid], 16, d)[1][1][0, slot, 1, 0] = float("nan")  # the step of dimensions 32 .. 63
        o[2:, :3, 32:] = float("nan")
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints([0, 5]).to(DEV), ints(total).to(DEV), table.to(DEV))
    within(got, o, paged_tolerance(o, spread, size, BF16, d, bits, total, 1.0))


def test_paged_attention_tiny_and_huge_steps():
    """Values of very different size in one cache: the weights p step keep their precision whatever the steps are."""
    hq, hkv, d, page = 3, 1, 64, 16
    for factor in (1e-6, 1.0, 3e4, 1e8):
        g = gen(31)
        k, v = torch.randn(90, hkv, d, generator=g).to(BF16), (torch.randn(90, hkv, d, generator=g) * factor).to(BF16)
        v[::7] = (v[::7].float() * 1e-3).to(BF16)
        table, n_pages = make_table([90], page)
        cache = ops.kv_cache(n_pages, page, hkv, d, 4, device="cpu")
        S.append(cache, page, k, v, [0, 90], [90], table)
        q = torch.randn(1, hq, d, generator=g).to(BF16)
        o, spread, size = paged_reference(q, cache, page, table, [1], [90])
        got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints([0, 1]).to(DEV), ints([90]).to(DEV), table.to(DEV))
        within(got, o, paged_tolerance(o, spread, size, BF16, d, 4, [90], factor))


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_attention_leaves_out_pages_that_do_not_exist(bits):
    """kv_len past the table and a page outside the cache: nothing outside is read, the error word tells, and sequences
    that are whole are right."""
    heads = (6, 2, 64)
    cache, table = filled_cache([40, 40, 40], heads, bits, 16, BF16, seed=4)
    q = torch.randn(3, 6, 64, generator=gen(5)).to(BF16)
    o, spread, size = paged_reference(q, cache, 16, table, [1, 1, 1], [40, 40, 40])
    broken = table.clone()
    broken[0, 1] = 1 << 20
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints([0, 1, 2, 3]).to(DEV), ints([40, 500, 40]).to(DEV),
                              broken.to(DEV))
    within(got[2:], o[2:], paged_tolerance(o, spread, size, BF16, 64, bits, [40], 1.0)[2:])
    assert L.device_error(reset=True) == L.ERR_BAD_PAGE


def test_paged_attention_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes, the sequence in its last pages."""
    heads, page, n = (3, 1, 64), 256, 300
    per = page * 80  # bytes
    n_pages = (1 << 32) // per + 10
    cache = torch.empty(n_pages, 1, page, 80, dtype=torch.uint8, device=DEV)
    small, table = filled_cache([n], heads, 4, page, BF16, seed=6)
    cache[-small.shape[0]:] = small.to(DEV)
    q = torch.randn(1, 3, 64, generator=gen(7)).to(BF16)
    o, spread, size = paged_reference(q, small, page, table, [1], [n])
    far = (table + (n_pages - small.shape[0])).to(DEV)
    got = ops.paged_attention(q.to(DEV), cache, ints([0, 1]).to(DEV), ints([n]).to(DEV), far)
    within(got, o, paged_tolerance(o, spread, size, BF16, 64, 4, [n], 1.0))
    k = torch.randn(1, 1, 64, generator=gen(8)).to(BF16)
    want = small.clone()
    S.append(want, page, k, k, [0, 1], [n + 1], table)
    ops.kv_append(cache, k.to(DEV), k.to(DEV), ints([0, 1]).to(DEV), ints([n + 1]).to(DEV), far)
    assert torch.equal(cache[-small.shape[0]:].cpu(), want)


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_attention_repeats_replays_and_other_streams(bits):
    heads, new, total = (15, 5, 64), [1, 1, 1], [900, 5, 333]
    cache, table = filled_cache(total, heads, bits, 16, BF16, seed=8, rest=0.5)
    q = torch.randn(3, 15, 64, generator=gen(9)).to(BF16).to(DEV)
    cache, table, cu, n = cache.to(DEV), table.to(DEV), ints(starts(new)).to(DEV), ints(total).to(DEV)
    ref = ops.paged_attention(q, cache, cu, n, table)
    assert all(torch.equal(ops.paged_attention(q, cache, cu, n, table), ref) for _ in range(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [ops.paged_attention(q, cache, cu, n, table) for _ in range(4)]
    mine = [ops.paged_attention(q, cache, cu, n, table) for _ in range(4)]  # overlaps with the other stream's calls
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, ref) for x in other + mine)
    # two graphs of the same call, each with a workspace of its own
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.paged_attention(q, cache, cu, n, table))
        graphs.append(graph)
    n.copy_(ints([600, 1, 20]))
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    now = ops.paged_attention(q, cache, cu, n, table)
    assert torch.equal(outs[0], now) and torch.equal(outs[1], now)


# ----------------------------------------------------------------------------- arguments

def test_arguments_that_do_not_fit_are_refused():
    q, kv = torch.zeros(4, 6, 64, dtype=BF16, device=DEV), torch.zeros(4, 2, 64, dtype=BF16, device=DEV)
    cu, n, table = ints([0, 4]).to(DEV), ints([4]).to(DEV), ints([[0]]).to(DEV)
    cache, wide = ops.kv_cache(1, 16, 2, 64), torch.zeros(1, 64, dtype=torch.int32, device=DEV)
    calls = [
        lambda: ops.packed_attention(q, kv.half(), kv.half(), cu),
        lambda: ops.packed_attention(q, kv, kv[:2], cu),
        lambda: ops.packed_attention(q.transpose(0, 1), kv, kv, cu),
        lambda: ops.packed_attention(q, kv, kv, cu.long()),
        lambda: ops.packed_attention(q, kv, kv, cu, cu[:1]),
        lambda: ops.packed_attention(q, kv, kv, cu, out=q[:3]),
        lambda: ops.packed_attention(q.float(), kv.float(), kv.float(), cu),
        lambda: ops.packed_attention(q[..., :48], kv[..., :48], kv[..., :48], cu),
        lambda: ops.kv_append(cache, kv, kv[:3], cu, n, table),
        lambda: ops.kv_append(cache, kv, kv, cu, n.long(), table),
        lambda: ops.kv_append(cache, kv, kv, cu, n, table, q=q[:2]),
        lambda: ops.kv_append(cache, kv, kv, cu, n, table, q_out=q),
        lambda: ops.kv_append(cache, kv, kv, cu, n, table, rope_cs=torch.zeros(4, 16, 2, device=DEV)),
        lambda: ops.kv_append(cache, kv, kv, cu, n, table, pos=cu),
        lambda: ops.kv_append(ops.kv_cache(1, 16, 3, 64), kv, kv, cu, n, table),
        lambda: ops.kv_append(ops.kv_cache(1, 16, 2, 128, 4), kv, kv, cu, n, table),
        lambda: ops.kv_append(cache.half(), kv, kv, cu, n, table),
        lambda: ops.kv_append(cache, kv, kv, cu, n, table.expand(2, 1)),
        lambda: ops.kv_append(cache, kv, kv, cu, n, table, k_out=kv[:1]),
        lambda: ops.paged_attention(q, cache[:, :, :1], cu, n, table),
        lambda: ops.paged_attention(q, cache, cu, n, table.long()),
        lambda: ops.paged_attention(q, cache, cu, n, table, workspace=torch.zeros(8, device=DEV)),
        lambda: ops.paged_attention(q, cache, cu, n, wide, workspace=torch.zeros(64, dtype=torch.uint8, device=DEV)),
    ]
    for i, call in enumerate(calls):
        with pytest.raises((ValueError, L.SvlaError)):
            call()
            pytest.fail(f"call {i} was taken")


def test_no_rows_give_nothing():
    q, kv = torch.zeros(0, 6, 64, dtype=BF16, device=DEV), torch.zeros(0, 2, 64, dtype=BF16, device=DEV)
    cu, n, table = ints([0, 0]).to(DEV), ints([4]).to(DEV), ints([[0]]).to(DEV)
    cache = ops.kv_cache(1, 16, 2, 64)
    assert ops.packed_attention(q, kv, kv, cu).shape == (0, 6, 64)
    assert ops.paged_attention(q, cache, cu, n, table).shape == (0, 6, 64)
    assert ops.kv_append(cache, kv, kv, cu, n, table, q=q).shape == (0, 6, 64)


@pytest.mark.parametrize("bits", [16, 4])
def test_custom_ops_are_the_functions(bits):
    """torch.ops.svla.*: schema, aliasing and shapes as registered, results as the functions give them."""
    hq, hkv, d, lens = 6, 2, 64, [20, 600, 1]
    table, n_pages = make_table(lens, 16, seed=31)
    x = torch.randn(sum(lens), hq + 2 * hkv, d, generator=gen(32)).to(BF16).to(DEV)
    q, k, v = (t.contiguous() for t in x.split([hq, hkv, hkv], 1))
    cu, n, table, cs = ints(starts(lens)).to(DEV), ints(lens).to(DEV), table.to(DEV), ops.rope_table_wide(600, 10000.0, DEV, d)
    cache, other = ops.kv_cache(n_pages, 16, hkv, d, bits), ops.kv_cache(n_pages, 16, hkv, d, bits)
    rotated = ops.kv_append(cache, k, v, cu, n, table, q=q, rope_cs=cs)
    assert torch.equal(torch.ops.svla.kv_append(other, k, v, cu, n, table, q, cs, None), rotated)
    assert torch.equal(other.view(torch.uint8), cache.view(torch.uint8))
    last, one = rotated[torch.tensor(lens).cumsum(0) - 1], ints([0, 1, 2, 3]).to(DEV)
    assert torch.equal(torch.ops.svla.packed_attention(q, k, v, cu, None, True, 0.0), ops.packed_attention(q, k, v, cu))
    assert torch.equal(torch.ops.svla.paged_attention(last, cache, one, n, table, 0.0),
                       ops.paged_attention(last, cache, one, n, table))
    for op, args in [(torch.ops.svla.packed_attention, (q, k, v, cu, None, True, 0.0)),
                     (torch.ops.svla.kv_append, (other, k, v, cu, n, table, q, cs, None)),
                     (torch.ops.svla.paged_attention, (last, cache, one, n, table, 0.0))]:
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


# ----------------------------------------------------------------------------- together

@pytest.mark.parametrize("bits", [16, 4])
def test_prompts_then_tokens_as_a_server_runs_them(bits):
    """Three prompts prefilled (rows appended, prompt attention over the rows as the cache holds them), then four steps of
    single tokens and one of three drafted ones, against dense attention in 64 bits over the cached entries."""
    hq, hkv, d, page, dtype = 15, 5, 64, 16, BF16
    lens, steps = [50, 1, 177], [[1, 1, 1]] * 4 + [[3, 3, 3]]
    final = [n + sum(s[b] for s in steps) for b, n in enumerate(lens)]
    table, n_pages = make_table(final, page, seed=11)
    table_d, cs = table.to(DEV), ops.rope_table_wide(max(final), 10000.0, DEV, d)
    cache = ops.kv_cache(n_pages, page, hkv, d, bits, dtype)
    g, have = gen(12), [0, 0, 0]
    for step, new in enumerate([lens] + steps):
        have = [h + n for h, n in zip(have, new)]
        x = torch.randn(sum(new), hq + 2 * hkv, d, generator=g).to(dtype).to(DEV)
        q, k, v = x.split([hq, hkv, hkv], 1)
        cu, n = ints(starts(new)).to(DEV), ints(have).to(DEV)
        if step == 0:
            q, k, v = ops.kv_append(cache, k, v, cu, n, table_d, q=q, rope_cs=cs, want_rows=True)
            got = ops.packed_attention(q, k, v, cu)
        else:
            q = ops.kv_append(cache, k, v, cu, n, table_d, q=q, rope_cs=cs)
            got = ops.paged_attention(q, cache, cu, n, table_d)
        o, spread, size = paged_reference(q.cpu(), cache.cpu(), page, table, new, have)
        tol = paged_tolerance(o, spread, size, dtype, d, bits, have, 1.0)
        if step == 0:  # the rows were rounded to bf16 once more than the cache: keys move the scores, values the sums
            unit = torch.finfo(dtype).eps / 2
            tol = S.attention_tolerance(o, spread, size, dtype, d) + unit * (1.02 * spread + 2.1 * size[..., None] * spread)
        within(got, o, tol, f"step {step}")
