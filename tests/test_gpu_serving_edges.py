"""The serving operators on the GPU where a masked, hidden, huge or missing entry could reach a row that must not know of
it: values at the types' limits, scores of -infinity, groups of very different size, pages that are not there.

Bars as in test_gpu_serving.py (oracle.serving.attention_tolerance), with the floors derived beside each test.
"""

import math

import pytest
import torch

from oracle import serving as S
from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops
from tests.test_gpu_serving import (BF16, DEV, FP16, KERNELS, _no_device_error, filled_cache, gen, ints,  # noqa: F401
                                    make_table, packed_inputs, packed_reference, paged_reference, paged_tolerance, starts, within)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- packed prompts

# every place of a key that the exponentials of a tile treat alike, and the tiles' borders
PLACES = list(range(0, 20)) + [32, 33, 63, 64, 80, 113, 127, 128, 129, 144]


@pytest.mark.parametrize("impl", KERNELS)
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(3, 1, 64), (4, 2, 128)], ids=str)
def test_packed_attention_hidden_values_at_the_limit_of_the_type(impl, heads, dtype):
    """One sequence per place of a value of the type's largest size: rows before it are as if it were not there."""
    hq, hkv, d, n = *heads, 145
    lens = [n] * len(PLACES)
    q, kv = packed_inputs(lens, lens, hq, hkv, d, dtype, seed=40)
    o, spread, size = packed_reference(q, kv, lens, lens, True)
    for i, j in enumerate(PLACES):
        kv[i * n + j, hkv:] = torch.finfo(dtype).max * (-1) ** i
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints(starts(lens)).to(DEV), impl=impl)
    tol = S.attention_tolerance(o, spread, size, dtype, d)
    for i, j in enumerate(PLACES):
        within(got[i * n:i * n + j], o[i * n:i * n + j], tol[i * n:i * n + j], f"place {j}")


@pytest.mark.parametrize("impl", KERNELS)
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(3, 1, 64), (4, 2, 128)], ids=str)
@pytest.mark.parametrize("gone", [1, 20, 150])
def test_packed_attention_scores_of_minus_infinity(impl, heads, dtype, gone):
    """The first `gone` keys' scores are -infinity: rows that see no other key give zeros, the others what the keys behind
    give."""
    hq, hkv, d, n = *heads, 200
    q, kv = packed_inputs([n], [n], hq, hkv, d, dtype, seed=41)
    q[..., 5] = q[..., 5].abs() + 0.5
    some, tail = torch.arange(n) >= gone, kv[gone:]
    o, spread, size = packed_reference(q, tail, [n], [n - gone], True)
    kv[:gone, :hkv, 5] = -math.inf
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints([0, n]).to(DEV), impl=impl)
    assert bool((got[:gone] == 0).all())
    within(got[some.to(DEV)], o[some], S.attention_tolerance(o, spread, size, dtype, d)[some])


@pytest.mark.parametrize("impl", KERNELS)
@pytest.mark.parametrize("heads", [(3, 1, 64), (4, 2, 128)], ids=str)
def test_packed_attention_small_weights_beside_a_large_one(impl, heads):
    """fp16: a first key with values of zero takes all but 2^-23.5 per key of the weight, and the rest of the weights make
    the result.  Their rounding is the type's down to 2^-21 of the largest (oracle tolerance); below, half a subnormal step,
    2^-25, of weights whose largest is 2^7 or more: 2^-32 of the largest for each key, times the largest value."""
    hq, hkv, d, n = *heads, 900
    q, kv = packed_inputs([n], [n], hq, hkv, d, FP16, seed=42)
    q[:] = 0
    q[..., 0] = 8.0
    kv[:, :hkv, 0] = 0
    kv[0, :hkv, 0] = 23.5 * math.log(2.0) * d ** 0.5 / 8.0
    kv[:, hkv:] = 1 + kv[:, hkv:].abs()
    kv[0, hkv:] = 0
    o, spread, size = packed_reference(q, kv, [n], [n], True)
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints([0, n]).to(DEV), impl=impl)
    floor = n * 2.0 ** -32 * float(kv[:, hkv:].max())
    # results of 1e-7 to 1e-3: the output's own half step is 2^-25 where it is subnormal
    within(got, o, S.attention_tolerance(o, spread, size, FP16, d, floor=floor + 2.0 ** -25))


@pytest.mark.parametrize("impl", KERNELS)
@pytest.mark.parametrize("heads", [(15, 5, 64), (8, 2, 128)], ids=str)
def test_packed_attention_one_long_prompt_among_many_short_ones(impl, heads):
    hq, hkv, d = heads
    lens = [5] * 60 + [1500] + [5] * 67
    q, kv = packed_inputs(lens, lens, hq, hkv, d, BF16, seed=43)
    o, spread, size = packed_reference(q, kv, lens, lens, True)
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints(starts(lens)).to(DEV), impl=impl)
    within(got, o, S.attention_tolerance(o, spread, size, BF16, d))


@pytest.mark.parametrize("impl", KERNELS)
def test_packed_attention_and_append_rows_beyond_32_bits(impl):
    """Rows 2^26 elements apart: the last ones lie behind 2^31 elements."""
    hq, hkv, d, n, page = 6, 2, 64, 40, 16
    q, kv = packed_inputs([n], [n], hq, hkv, d, BF16, seed=44)
    o, spread, size = packed_reference(q, kv, [n], [n], True)
    far = torch.empty(n, 1 << 20, d, dtype=BF16, device=DEV)
    x, out = far[:, :hq + 2 * hkv], far[:, 20:20 + hq]
    x.copy_(torch.cat([q, kv], 1))
    qd, kd, vd = x.split([hq, hkv, hkv], 1)
    got = ops.packed_attention(qd, kd, vd, ints([0, n]).to(DEV), out=out, impl=impl)
    within(got, o, S.attention_tolerance(o, spread, size, BF16, d))
    table, n_pages = make_table([n], page)
    cache = ops.kv_cache(n_pages, page, hkv, d, 4, device=DEV)
    want = cache.cpu().clone()
    cs = ops.rope_table_wide(n, 10000.0, DEV, d)
    rq, rk, rv = S.append(want, page, kv[:, :hkv], kv[:, hkv:], [0, n], [n], table, cs.cpu(), None, q)
    ops.kv_append(cache, kd, vd, ints([0, n]).to(DEV), ints([n]).to(DEV), table.to(DEV), q=qd, rope_cs=cs, q_out=qd, k_out=kd,
                  v_out=vd)
    assert torch.equal(cache.cpu(), want) and torch.equal(x.cpu(), torch.cat([rq, rk, rv], 1))


# ----------------------------------------------------------------------------- paged attention

def step_floor(q, cache, page, table, new, total):
    """4 bits: what rounding the weights p step to fp16 can lose below its normal range, [rows, heads, D].

    A warp keeps the weights of every group of 32 dimensions at a power of two of their own, such that the largest it has
    met is 2^2 or more; a smaller one is off by half a subnormal step, 2^-25, that is by 2^-27 of the largest, times a code
    of at most 15, for each entry."""
    d, at, out = q.shape[2], starts(new), []
    g = q.shape[1] // cache.shape[1]
    for b in range(len(new)):
        k = S.rows(cache, page, d, table[b], total[b])[0]
        pairs = [S.split4(cache[int(table[b, n // page])], page, d)[1][1][:, n % page, :, 0] for n in range(total[b])]
        step = torch.stack(pairs).double().abs()  # [entries, hkv, d / 32]
        for i, n in enumerate(S.causal_seen(new[b], total[b])):
            row = torch.zeros(q.shape[1], d, dtype=torch.float64)
            for h in range(q.shape[1] if n else 0):
                p = torch.softmax(k[:n, h // g] @ q[at[b] + i, h].double() * d ** -0.5, 0)
                row[h] = (p[:, None] * step[:n, h // g]).amax(0).repeat_interleave(32)
            out.append(row * n * 15 * 2.0 ** -27)
    return torch.stack(out)


def check_groups(q, cache, page, table, new, total, what):
    d = q.shape[2]
    o, spread, size = paged_reference(q, cache, page, table, new, total)
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints(starts(new)).to(DEV), ints(total).to(DEV), table.to(DEV))
    tol = S.attention_tolerance(o, spread, size, q.dtype, d, weight_unit=2.0 ** -11)
    within(got, o, tol + step_floor(q, cache, page, table, new, total), what)


def cache_of(k, v, page, width=None, seed=50):
    table, n_pages = make_table([k.shape[0]], page, seed, width=width)
    cache = ops.kv_cache(n_pages, page, k.shape[1], k.shape[2], 4, k.dtype, device="cpu")
    S.append(cache, page, k, v, [0, k.shape[0]], [k.shape[0]], table)
    return cache, table


@pytest.mark.parametrize("heads", [(3, 1, 64), (15, 5, 64), (8, 2, 128), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("new,n,width", [(1, 200, None), (5, 333, None), (1, 1500, 100), (3, 1500, 100)])
@pytest.mark.parametrize("factor", [1e4, 1e6, 1e-6])
def test_paged_attention_groups_of_very_different_size(heads, new, n, width, factor):
    """One group of dimensions `factor` times the others: each is as precise as if it were alone."""
    hq, hkv, d = heads
    g = gen(51)
    k, v = (torch.randn(n, hkv, d, generator=g) for _ in range(2))
    v[..., 32:64] *= factor
    cache, table = cache_of(k.to(BF16), v.to(BF16), 16, width)
    q = torch.randn(new, hq, d, generator=g).to(BF16)
    check_groups(q, cache, 16, table, [new], [n], f"factor {factor}")


@pytest.mark.parametrize("heads", [(3, 1, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("new,n,width", [(1, 200, None), (5, 333, None), (3, 1500, 100)])
@pytest.mark.parametrize("factor,score,at", [(1e4, -30.0, 0), (1e6, -40.0, 77), (1e6, -40.0, 190), (1e9, -60.0, 3)])
def test_paged_attention_large_value_at_a_low_score(heads, new, n, width, factor, score, at):
    """One entry's values are `factor` times the others' and its weight next to nothing: the others keep their precision."""
    hq, hkv, d = heads
    g = gen(52)
    k, v = (torch.randn(n, hkv, d, generator=g) for _ in range(2))
    q = torch.randn(new, hq, d, generator=g)
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[at, :, 0] = score * d ** 0.5 / 4.0
    v[at] *= factor
    cache, table = cache_of(k.to(BF16), v.to(BF16), 16, width)
    check_groups(q.to(BF16), cache, 16, table, [new], [n], f"entry {at}")


@pytest.mark.parametrize("heads", [(3, 1, 64), (8, 2, 128)], ids=str)
def test_paged_attention_growing_and_shrinking_steps_and_scores(heads):
    """Scores that rise along the sequence while the values' steps fall, and the other way round: maxima and exponents
    move all the time."""
    hq, hkv, d, n = *heads, 1500
    for way, rise in ((1, 60.0), (-1, 60.0), (1, 400.0)):
        g = gen(53)
        k, v = (torch.randn(n, hkv, d, generator=g) for _ in range(2))
        q = torch.randn(2, hq, d, generator=g)
        q[..., 0] = 4.0
        k[..., 0] = (torch.linspace(0, rise, n) * d ** 0.5 / 4.0)[:, None]
        v *= torch.logspace(-12 * way, 12 * way, n).flip(0)[:, None, None]
        v[..., 32:64] *= torch.logspace(6, -6, n)[:, None, None]
        for width in (None, 120):
            cache, table = cache_of(k.to(BF16), v.to(BF16), 16, width)
            check_groups(q.to(BF16), cache, 16, table, [2], [n], f"way {way} rise {rise}")


@pytest.mark.parametrize("heads", [(15, 5, 64), (32, 8, 128)], ids=str)
@pytest.mark.parametrize("new,n", [(1, 1), (1, 2), (1, 7), (3, 40), (1, 300)])
def test_paged_attention_fp16_weights_keep_the_rest_of_their_rounding(heads, new, n):
    """4 bits, fp16: a weight p step is two fp16 numbers, off by 2^-22 of itself.  The bar is attention_tolerance with that,
    and the output's own rounding."""
    hq, hkv, d = heads
    g = gen(65)
    k, v = (torch.randn(n, hkv, d, generator=g) for _ in range(2))
    cache, table = cache_of(k.half(), v.half(), 16)
    q = torch.randn(new, hq, d, generator=g).half()
    o, spread, size = paged_reference(q, cache, 16, table, [new], [n])
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints([0, new]).to(DEV), ints([n]).to(DEV), table.to(DEV))
    tol = S.attention_tolerance(o, spread, size, FP16, d, weight_unit=2.0 ** -22)
    within(got, o, tol + step_floor(q, cache, 16, table, [new], [n]))


@pytest.mark.parametrize("heads", [(3, 1, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("n", [1, 2, 33, 65, 130])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_paged_attention_non_finite_group_leaves_the_others(heads, n, bad, dtype):
    """4 bits, an infinity or a NaN in the last entry's values: its group of 32 dimensions is NaN, the others are right."""
    hq, hkv, d = heads
    g = gen(54)
    k, v = (torch.randn(n, hkv, d, generator=g) for _ in range(2))
    q = torch.randn(1, hq, d, generator=g).to(dtype)
    v[n - 1, :, 40] = bad
    for width in (None, 64):
        cache, table = cache_of(k.to(dtype), v.to(dtype), 16, width)
        check_groups(q, cache, 16, table, [1], [n], f"{n} entries")


@pytest.mark.parametrize("heads", [(3, 1, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("new", [1, 3])
def test_paged_attention_small_weights_beside_a_large_one(heads, new):
    """16 bits, fp16, as for packed prompts above: the floor is 2^-32 of the largest weight for each entry."""
    hq, hkv, d, n, page = *heads, 900, 16
    g = gen(61)
    k, v = (torch.randn(n, hkv, d, generator=g) for _ in range(2))
    k[..., 0], k[0, :, 0] = 0, 23.5 * math.log(2.0) * d ** 0.5 / 8.0
    v = 1 + v.abs()
    v[0] = 0
    q = torch.zeros(new, hq, d, dtype=FP16)
    q[..., 0] = 8.0
    table, n_pages = make_table([n], page, 62)
    cache = ops.kv_cache(n_pages, page, hkv, d, 16, FP16, device="cpu")
    S.append(cache, page, k.half(), v.half(), [0, n], [n], table)
    o, spread, size = paged_reference(q, cache, page, table, [new], [n])
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints([0, new]).to(DEV), ints([n]).to(DEV), table.to(DEV))
    within(got, o, S.attention_tolerance(o, spread, size, FP16, d, floor=n * 2.0 ** -32 * float(v.max()) + 2.0 ** -25))


@pytest.mark.parametrize("heads", [(3, 1, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("gone,total,width", [(2, 5, None), (40, 45, None), (1500, 2000, 200), (2000, 2003, 200)])
def test_paged_attention_scores_of_minus_infinity(heads, gone, total, width):
    """16 bits, the first `gone` entries' scores are -infinity: what rows see behind them, or zeros."""
    hq, hkv, d = heads
    new, page = 5, 16
    cache, table = filled_cache([total], heads, 16, page, BF16, seed=55, width=width)
    q = torch.randn(new, hq, d, generator=gen(56)).to(BF16)
    q[..., 5] = q[..., 5].abs() + 0.5
    k, v = S.rows(cache, page, d, table[0], total)[:2]
    o, spread, size = S.attend_dense(q.double(), k[gone:], v[gone:], S.causal_seen(new, total - gone), d ** -0.5)
    for n in range(gone):
        cache[int(table[0, n // page]), :, 0, n % page, 5] = -math.inf
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints([0, new]).to(DEV), ints([total]).to(DEV), table.to(DEV))
    none = [i for i in range(new) if total - new + i < gone]
    assert bool((got[none] == 0).all())
    within(got, o, S.attention_tolerance(o, spread, size, BF16, d))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("batch", [127, 128, 129, 300])
@pytest.mark.parametrize("width", [None, 100], ids=["one piece", "pieces"])
def test_paged_attention_finds_every_item_of_many_sequences(bits, batch, width):
    """Sequences without tokens, with one and with several, with nothing cached before and with up to 70 entries."""
    hq, hkv, d, page = 3, 1, 64, 16
    new = [(1, 0, 1, 2, 1, 9)[(i * i + i // 7) % 6] for i in range(batch)]
    total = [n + (i * 31) % 70 for i, n in enumerate(new)]
    cache, table = filled_cache(total, (hq, hkv, d), bits, page, BF16, seed=66, width=width)
    q = torch.randn(sum(new), hq, d, generator=gen(67)).to(BF16)
    o, spread, size = paged_reference(q, cache, page, table, new, total)
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints(starts(new)).to(DEV), ints(total).to(DEV), table.to(DEV))
    within(got, o, paged_tolerance(o, spread, size, BF16, d, bits, total, 1.0))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("width", [None, 64], ids=["one piece", "pieces"])
def test_paged_attention_rows_whose_pages_are_missing(bits, width):
    """What is readable counts, and where nothing is, zeros: a page outside the cache in the middle, all pages outside, a
    sequence longer than its table (three drafted tokens, all of which see all that the table reaches)."""
    hq, hkv, d, page = 6, 2, 64, 16
    heads, lens, new = (hq, hkv, d), [40, 20, 48, 40], [2, 1, 3, 1]
    cache, table = filled_cache(lens, heads, bits, page, BF16, seed=57, width=width)
    q = torch.randn(sum(new), hq, d, generator=gen(58)).to(BF16)
    broken, at = table.clone(), starts(new)
    broken[0, 1], broken[1, :2] = 1 << 20, -1
    total = [40, 20, 500, 40]
    if width is not None:
        broken = broken.clone()
        total[2] = 48 + 2  # the table is wide: two entries that it does not name
        broken[2, 3] = -1
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints(at).to(DEV), ints(total).to(DEV), broken.to(DEV))
    assert L.device_error(reset=True) == L.ERR_BAD_PAGE
    assert bool((got[at[1]:at[2]] == 0).all())
    for b, keep, seen in ((0, [n for n in range(40) if n // page != 1], [23, 24]),
                          (2, list(range(48)), [48] * 3), (3, list(range(40)), [40])):
        k, v, ks, vs = S.rows(cache, page, d, table[b], lens[b])
        o, spread, size = S.attend_dense(q[at[b]:at[b + 1]].double(), k[keep], v[keep], seen, d ** -0.5, ks[keep], vs[keep])
        within(got[at[b]:at[b + 1]], o, paged_tolerance(o, spread, size, BF16, d, bits, [lens[b]], 1.0), f"sequence {b}")


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_attention_limit_counts_entries_past_the_table(bits):
    """Three drafted tokens of a sequence that is two entries longer than its table: the first sees all the table holds, as
    do the others."""
    heads, page = (6, 2, 64), 16
    cache, table = filled_cache([48], heads, bits, page, BF16, seed=59)
    q = torch.randn(1, 6, 64, generator=gen(60)).to(BF16).expand(3, 6, 64).contiguous()
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints([0, 3]).to(DEV), ints([50]).to(DEV), table.to(DEV))
    assert L.device_error(reset=True) == L.ERR_BAD_PAGE
    k, v, ks, vs = S.rows(cache, page, 64, table[0], 48)
    o, spread, size = S.attend_dense(q.double(), k, v, [48] * 3, 0.125, ks, vs)
    within(got, o, paged_tolerance(o, spread, size, BF16, 64, bits, [48], 1.0))


# ----------------------------------------------------------------------------- appending

@pytest.mark.parametrize("heads", [(2, 64), (2, 128)], ids=str)
def test_kv_append_of_groups_with_an_offset_or_a_huge_range(heads):
    """4 bits: bytes and rows as the same fp32 operations give them, with an offset beside the range and a range beyond
    fp32's largest number."""
    hkv, d, n, page = *heads, 40, 16
    k = torch.rand(n, hkv, d, generator=gen(63)) + torch.tensor([100.0, -100.0, 1000.0, 0.0]).repeat(n // 4)[:, None, None]
    k, v = k.to(BF16), (k.flip(0) * 3).to(BF16)
    v[7, 0, 0], v[7, 0, 1] = -3e38, 3e38
    table, n_pages = make_table([n], page, 64)
    cache = ops.kv_cache(n_pages, page, hkv, d, 4, device=DEV)
    want = cache.cpu().clone()
    _, rk, rv = S.append(want, page, k, v, [0, n], [n], table)
    _, gk, gv = ops.kv_append(cache, k.to(DEV), v.to(DEV), ints([0, n]).to(DEV), ints([n]).to(DEV), table.to(DEV), want_rows=True)
    assert torch.equal(cache.cpu(), want)
    assert torch.equal(gk.cpu(), rk)
    nan = torch.isnan(rv)
    assert bool(nan[7, 0, :32].all()) and int(nan.sum()) == 32
    assert torch.equal(torch.isnan(gv).cpu(), nan) and torch.equal(gv.cpu()[~nan], rv[~nan])


# ----------------------------------------------------------------------------- arguments

def test_scales_that_do_not_fit_are_refused():
    q, kv = torch.zeros(4, 6, 64, dtype=BF16, device=DEV), torch.zeros(4, 2, 64, dtype=BF16, device=DEV)
    cu, n, table = ints([0, 4]).to(DEV), ints([4]).to(DEV), ints([[0]]).to(DEV)
    cache = ops.kv_cache(1, 16, 2, 64)
    for scale in (-0.125, math.inf, -math.inf, math.nan, 1e-60, 1e60):
        for call in (lambda: ops.packed_attention(q, kv, kv, cu, scale=scale),
                     lambda: ops.paged_attention(q, cache, cu, n, table, scale=scale)):
            with pytest.raises((ValueError, L.SvlaError), match="scale"):
                call()


def test_rotation_table_without_positions_is_refused():
    kv = torch.zeros(4, 2, 64, dtype=BF16, device=DEV)
    with pytest.raises((ValueError, L.SvlaError), match="rope_cs"):
        ops.kv_append(ops.kv_cache(1, 16, 2, 64), kv, kv, ints([0, 4]).to(DEV), ints([4]).to(DEV), ints([[0]]).to(DEV),
                      rope_cs=torch.zeros(0, 32, 2, device=DEV))
