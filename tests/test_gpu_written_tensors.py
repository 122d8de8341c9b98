"""Tensors that a caller gives to be written have a new version afterwards, so a graph that saved one refuses to go on."""

import pytest
import torch

from smolvla_mujoco_libero_b200 import ops

pytestmark = pytest.mark.gpu
DEV, BF16 = "cuda", torch.bfloat16


def calls():
    """(name, call, the tensors that it writes)"""
    g = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g).to(BF16).to(DEV)  # noqa: E731
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    x, res, values = rand(4, 64), rand(4, 64), rand(4, 64)
    codes, scale = torch.zeros(4, 64, dtype=torch.int8, device=DEV), torch.zeros(4, device=DEV)
    w, ws = ops.pack_weight_i8(rand(64, 64))
    out, logits, u = rand(4, 64), rand(4, 64), torch.full((4,), 0.5, device=DEV)
    tokens, logprob = ints(0, 0, 0, 0), torch.zeros(4, device=DEV)
    q, k, v = rand(4, 3, 64), rand(4, 1, 64), rand(4, 1, 64)
    cache, cu, n, table = rand(2, 1, 2, 16, 64), ints(0, 4), ints(4), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    q_out, k_out, v_out, o1, o2 = rand(4, 3, 64), rand(4, 1, 64), rand(4, 1, 64), rand(4, 3, 64), rand(4, 3, 64)
    return [
        ("quantize_rows", lambda: ops.quantize_rows(x, residual=res, sum=res, codes=codes, scale=scale, values=values), [res, codes, scale, values]),
        ("linear_i8_rows", lambda: ops.linear_i8_rows(codes, scale, w, ws, residual=out, out=out), [out]),
        ("sample_tokens", lambda: ops.sample_tokens(logits, u, tokens=tokens, logprob=logprob), [tokens, logprob]),
        ("kv_append", lambda: ops.kv_append(cache, k, v, cu, n, table, q=q, q_out=q_out, k_out=k_out, v_out=v_out), [cache, q_out, k_out, v_out]),
        ("packed_attention", lambda: ops.packed_attention(q, k, v, cu, out=o1), [o1]),
        ("paged_attention", lambda: ops.paged_attention(q, cache, cu, n, table, out=o2), [o2]),
    ]


@pytest.mark.parametrize("i", range(6), ids=["quantize_rows", "linear_i8_rows", "sample_tokens", "kv_append", "packed_attention", "paged_attention"])
def test_written_tensors_have_a_new_version(i):
    _, call, tensors = calls()[i]
    before = [t._version for t in tensors]
    call()
    assert all(t._version > b for t, b in zip(tensors, before))
    with torch.inference_mode():  # tensors without versions
        calls()[i][1]()


def test_a_graph_notices_what_it_saved():
    leaf = torch.randn(4, 64, device=DEV, dtype=BF16, requires_grad=True)
    h = leaf * 2
    loss = h.square().sum()
    with torch.no_grad():
        ops.quantize_rows(torch.ones(4, 64, device=DEV, dtype=BF16), residual=h, sum=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
