"""Operands that torch calls contiguous and no kernel can read as they are: packed ones two bytes into a buffer, and single
rows of odd strides.  Each gives the bits of its aligned copy."""

from __future__ import annotations

import pytest
import torch

from streamindex_amd import (chunked_indexer_topk, flash_hca_forward, indexer_topk_q, paged_attn_fwd, quant, sparse_attn_bwd,
                             sparse_attn_fwd, sparse_attn_fwd_kv2, synth)

pytestmark = pytest.mark.gpu


def shifted(t):
    """A packed copy one element into a buffer."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = buf[1:].view(t.shape)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out


def one_of_odd_rows(t):
    """A copy of a tensor of one row whose (unused) strides are odd."""
    wide = torch.empty(*t.shape[:-1], t.shape[-1] + 1, dtype=t.dtype, device=t.device)
    out = wide[..., :-1]
    out.copy_(t)
    assert out.is_contiguous() and out.stride(0) % 8
    return out


def same(got, want):
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def rand(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,H,place", [(3, 4, shifted), (1, 1, shifted), (1, 1, one_of_odd_rows)])
def test_paged_attn(N, H, place, dtype):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q, kv = rand(N, H, 64, dtype=dtype), rand(5, 16, 64, dtype=dtype, seed=1)
    args = (kv, i32([[3, 0, 4]]), i32([0, N]), i32([40]), torch.zeros(H, device="cuda"))
    same(paged_attn_fwd(place(q), *args), paged_attn_fwd(q, *args))


@pytest.mark.parametrize("B,S,H,place", [(2, 5, 16, shifted), (1, 1, 1, shifted), (1, 1, 1, one_of_odd_rows)])
def test_sparse_attn(B, S, H, place):
    q, kv, kv2 = rand(B, S, H, 64), rand(B, 9, 64, seed=1), rand(B, 7, 64, seed=2)
    sink = torch.zeros(H, device="cuda")
    idx = torch.arange(8, device="cuda", dtype=torch.int32).expand(B, S, 8).contiguous()
    o, lse = sparse_attn_fwd(q, kv, sink, idx)
    same(sparse_attn_fwd(place(q), shifted(kv), sink, idx), (o, lse))
    same(sparse_attn_fwd_kv2(place(q), shifted(kv), shifted(kv2), sink, idx), sparse_attn_fwd_kv2(q, kv, kv2, sink, idx))
    do = rand(B, S, H, 64, seed=3)
    same(sparse_attn_bwd(place(q), shifted(kv), sink, idx, place(o), lse, place(do)),
         sparse_attn_bwd(q, kv, sink, idx, o, lse, do))


@pytest.mark.parametrize("S,H", [(40, 16), (256, 64)])
def test_hca(S, H):
    D, m = 64, 8
    q, kv, comp, do = rand(1, S, H, D), rand(1, S, D, seed=1), rand(1, S // m, D, seed=2), rand(1, S, H, D, seed=3)
    out = []
    for place in (lambda t: t, shifted):
        leaves = [place(t).detach().requires_grad_() for t in (q, kv, comp)]
        sink = torch.zeros(H, device="cuda", requires_grad=True)
        o = flash_hca_forward(*leaves, sink, n_win=16, m_prime=m)
        o.backward(place(do))
        out.append([o, *(t.grad for t in leaves), sink.grad])
    same(*out)


@pytest.mark.parametrize("S,place", [(64, shifted), (1, shifted), (1, one_of_odd_rows)])
def test_indexer(S, place):
    q, k, w = synth.indexer_inputs(1, S, 1 if S == 1 else 16, 128, T=32, seed=5)
    same(chunked_indexer_topk(place(q), shifted(k), w, 8), chunked_indexer_topk(q, k, w, 8))


def test_quantised_indexer():
    q, k, w = synth.indexer_inputs(1, 64, 16, 128, ratio=4, seed=5)
    q4, qs = quant.fp4_act_quant(q, 32)
    k8, ks = quant.act_quant(k, 128)
    same(indexer_topk_q(shifted(q4), qs, shifted(k8.view(torch.uint8)).view(k8.dtype), ks, w, 8),
         indexer_topk_q(q4, qs, k8, ks, w, 8))
