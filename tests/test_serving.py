"""CPU checks of the serving operators: what the C ABI and the torch layer refuse before any launch, the descriptors'
layouts, and the 64-bit plain forms that the GPU tests compare with."""

import ctypes

import pytest
import torch

from oracle import serving as S
from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops
from tests.test_capi import _c_sizeof


@pytest.mark.parametrize("cname,pyname", [("svla_kv_append_desc", "KvAppendDesc"),
                                          ("svla_packed_attn_desc", "PackedAttnDesc"),
                                          ("svla_paged_attn_desc", "PagedAttnDesc")])
def test_struct_layouts(cname, pyname, tmp_path):
    assert ctypes.sizeof(getattr(L, pyname)) == _c_sizeof(cname, tmp_path)


# Addresses that are never read: every case below is refused on the host.
def _append(**kw):
    d = L.KvAppendDesc()
    d.q, d.k, d.v, d.q_out, d.cache = 0x100000, 0x200000, 0x300000, 0x400000, 0x500000
    d.cu_q, d.kv_len, d.page_table = 0x600000, 0x700000, 0x800000
    d.q_rs, d.k_rs, d.v_rs, d.q_out_rs, d.page_table_rs = 960, 320, 320, 960, 4
    d.batch, d.total_q, d.hq, d.hkv, d.head_dim, d.dtype = 1, 1, 15, 5, 64, L.DT_BF16
    d.bits, d.page_size, d.n_pages, d.max_pages = 16, 16, 8, 4
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _packed(**kw):
    d = L.PackedAttnDesc()
    d.q, d.k, d.v, d.o, d.cu_q, d.cu_k = 0x100000, 0x200000, 0x300000, 0x400000, 0x500000, 0x600000
    d.q_rs, d.k_rs, d.v_rs, d.o_rs = 960, 320, 320, 960
    d.batch, d.total_q, d.total_k, d.hq, d.hkv, d.head_dim, d.dtype, d.causal = 1, 4, 4, 15, 5, 64, L.DT_BF16, 1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _paged(**kw):
    d = L.PagedAttnDesc()
    d.q, d.cache, d.o, d.cu_q, d.kv_len, d.page_table = 0x100000, 0x200000, 0x300000, 0x400000, 0x500000, 0x600000
    d.workspace, d.workspace_bytes = 0x700000, 1 << 30
    d.q_rs, d.o_rs, d.page_table_rs = 960, 960, 64
    d.batch, d.total_q, d.hq, d.hkv, d.head_dim, d.dtype = 1, 1, 15, 5, 64, L.DT_BF16
    d.bits, d.page_size, d.n_pages, d.max_pages = 4, 16, 80, 64
    for k, v in kw.items():
        setattr(d, k, v)
    return d


REFUSED = [
    ("svla_kv_append", _append, dict(hkv=4), "multiple"),
    ("svla_kv_append", _append, dict(head_dim=96), "head_dim"),
    ("svla_kv_append", _append, dict(dtype=L.DT_FLOAT), "dtype"),
    ("svla_kv_append", _append, dict(bits=8), "bits"),
    ("svla_kv_append", _append, dict(page_size=24), "page_size"),
    ("svla_kv_append", _append, dict(page_size=512), "page_size"),
    ("svla_kv_append", _append, dict(n_pages=0), "n_pages"),
    ("svla_kv_append", _append, dict(page_table_rs=3), "page_table"),
    ("svla_kv_append", _append, dict(k=0x200002), "k must be 16-byte"),
    ("svla_kv_append", _append, dict(v_rs=316), "v must be"),
    ("svla_kv_append", _append, dict(q_rs=952), "q must be"),
    ("svla_kv_append", _append, dict(q_out=None), "q_out is null"),
    ("svla_kv_append", _append, dict(k_out=0x900008, k_out_rs=320), "k_out must be"),
    ("svla_kv_append", _append, dict(rope_cs=0x900000, max_pos=0), "rope_cs"),
    ("svla_kv_append", _append, dict(cache=0x500008), "cache must be"),
    ("svla_kv_append", _append, dict(kv_len=None), "null"),
    ("svla_kv_append", _append, dict(batch=-1), "negative"),
    ("svla_packed_attention", _packed, dict(hq=16), "multiple"),
    ("svla_packed_attention", _packed, dict(hq=65, hkv=1, q_rs=4160, o_rs=4160), "at most"),
    ("svla_packed_attention", _packed, dict(head_dim=80), "head_dim"),
    ("svla_packed_attention", _packed, dict(dtype=L.DT_INT32), "dtype"),
    ("svla_packed_attention", _packed, dict(cu_k=None), "cu_k"),
    ("svla_packed_attention", _packed, dict(q_rs=964), "q must be"),
    ("svla_packed_attention", _packed, dict(o=None), "o is null"),
    ("svla_packed_attention", _packed, dict(k_rs=0), "k must be"),
    ("svla_packed_attention", _packed, dict(total_k=-1), "negative"),
    ("svla_paged_attention", _paged, dict(hkv=0), "multiple"),
    ("svla_paged_attention", _paged, dict(bits=5), "bits"),
    ("svla_paged_attention", _paged, dict(page_size=8), "page_size"),
    ("svla_paged_attention", _paged, dict(workspace=None), "workspace"),
    ("svla_paged_attention", _paged, dict(workspace=0x700010), "workspace"),
    ("svla_paged_attention", _paged, dict(workspace_bytes=64), "workspace"),
    ("svla_paged_attention", _paged, dict(o_rs=8), "o must be"),
    ("svla_paged_attention", _paged, dict(q=0x100004), "q must be"),
    ("svla_paged_attention", _paged, dict(page_table=None), "null"),
]


@pytest.mark.parametrize("name,make,change,word", REFUSED)
def test_refused_before_any_launch(name, make, change, word):
    lib = L.lib()
    assert getattr(lib, name)(ctypes.byref(make(**change)), None) == 1
    assert word in lib.svla_last_error().decode(), lib.svla_last_error()


def test_null_descriptors_and_nothing_to_do():
    lib = L.lib()
    for name, make in (("svla_kv_append", _append), ("svla_packed_attention", _packed), ("svla_paged_attention", _paged)):
        assert getattr(lib, name)(None, None) == 1
        assert getattr(lib, name)(ctypes.byref(make(total_q=0)), None) == 0  # no rows: nothing is launched
        assert getattr(lib, name)(ctypes.byref(make(batch=0)), None) == 0
    assert lib.svla_rope_table_wide(None, 4, 64, 1e4, None) == 1
    assert lib.svla_rope_table_wide(0x100000, 4, 63, 1e4, None) == 1
    assert lib.svla_paged_attention_workspace_size(0, 1, 15, 5, 64, 4096) == 0
    assert lib.svla_paged_attention_workspace_size(1, 1, 15, 5, 64, 256) == 0  # short: no second launch, no workspace
    assert lib.svla_paged_attention_workspace_size(1, 1, 15, 5, 64, 4096) > 0


def test_cpu_tensors_are_refused():
    q, kv = torch.zeros(2, 15, 64, dtype=torch.bfloat16), torch.zeros(2, 5, 64, dtype=torch.bfloat16)
    cu, n = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    cache = ops.kv_cache(1, 16, 5, 64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.packed_attention(q, kv, kv, cu)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_append(cache, kv, kv, cu, n, table)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q, cache, cu, n, table)
    for bad in (dict(bits=8), dict(page_size=24), dict(head_dim=96), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            ops.kv_cache(**(dict(n_pages=1, page_size=16, kv_heads=1, head_dim=64, device="cpu") | bad))


def test_cache_shapes():
    assert ops.kv_cache(3, 32, 5, 64, device="cpu").shape == (3, 5, 2, 32, 64)
    c = ops.kv_cache(3, 32, 5, 128, bits=4, device="cpu")
    assert c.shape == (3, 5, 32, 160) and c.dtype == torch.uint8


def test_plain_quantisation_is_within_half_a_step():
    """low + step code is off by at most half a step, plus what rounding the pair to bf16 (2^-8 of its size, half a step
    of the type) takes from the ends: |low| 2^-8 at the lower end, and 15 steps of 2^-8 + |low| 2^-8 at the upper."""
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(3)) * 3
    codes, step, low = S.quantise(x)
    assert int(codes.max()) <= 15
    err = (S.held(codes, step, low) - x).abs().unflatten(-1, (-1, 32))
    s, m = step.float().unsqueeze(-1), low.float().abs().unsqueeze(-1)
    assert bool((err <= s * (0.5 + 15 * 2.0 ** -8) + m * 2.0 ** -8 + 1e-6).all())
    assert torch.equal(S.unpack4(S.pack4(codes)), codes)
    flat = torch.full((1, 64), 2.5)
    assert torch.equal(S.held(*S.quantise(flat)), flat)


def test_plain_attention_forms_agree():
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(n, h, 64, generator=g, dtype=torch.float64) for n, h in ((7, 6), (5, 2), (5, 2)))
    seen = S.causal_seen(7, 5)
    assert seen == [0, 0, 1, 2, 3, 4, 5]
    for a, b in zip(S.attend(q, k, v, seen, 0.125), S.attend_dense(q, k, v, seen, 0.125)):
        assert torch.allclose(a, b, atol=1e-12)
