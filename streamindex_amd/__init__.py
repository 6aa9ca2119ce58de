"""StreamIndex for MI355X: the DeepSeek-V4 CSA hot path on gfx950.

Operators (hand-written HIP kernels behind the C ABI in
``include/streamindex.h``, loaded from ``streamindex_amd/lib/libstreamindex.so``):

* :func:`chunked_indexer_topk` — fused lightning-indexer score + exact top-k;
* :func:`indexer_score`, :func:`indexer_score_topk`;
* :func:`indexer_topk_q`, :func:`chunked_indexer_topk_quantized` — the indexer over fp4
  queries and fp8 keys (the production V4 indexer dtypes), and
  ``streamindex_amd.quant`` / ``streamindex_amd.compressor`` for the quantisers and the
  token compressor;
* :func:`sparse_attn_fwd`, :func:`sparse_attn_bwd`, :func:`sparse_attn` — MQA sparse attention
  with sink, its backward and the autograd wrapper;
* :func:`flash_csa_forward`, :func:`build_csa_topk_idxs`, :func:`csa_topk_idxs` —
  the CSA composition (fused indexer → window + compressed index rows → attention);
* :func:`flash_hca_forward`, :func:`build_hca_topk_idxs` — HCA (window + every
  legal compressed entry);
* :func:`paged_plan`, :func:`paged_write`, :func:`paged_compress`, :func:`paged_attn_fwd` — serving steps over a paged
  cache, and :func:`flash_hca_paged_forward`, an HCA layer of them;
* :func:`paged_write_q`, :func:`paged_attn_q_fwd` — write and attention over a cache held in 8 bits;
* :func:`rotary`, :func:`norm_rotary` — rotary positions of the heads' rows, alone and behind their norm, with gradients, and
  :func:`rotary_freqs`.

The same names are importable under the reference's module paths through the
``flash_sparse`` package (``flash_sparse.triton.chunked_indexer`` etc.).
"""

from .indexer import (chunked_indexer_topk, chunked_indexer_topk_quantized, indexer_score, indexer_score_topk,
                      indexer_topk_q)
from .sparse_attn import (build_inverted_topk, sparse_attn, sparse_attn_bwd, sparse_attn_bwd_v2, sparse_attn_fwd,
                          sparse_attn_fwd_kv2, sparse_attn_kv2)
from .csa import build_csa_topk_idxs, csa_topk_idxs, flash_csa_forward
from .hca import build_hca_topk_idxs, flash_hca_forward, flash_hca_paged_forward
from .rotary import norm_rotary, rotary, rotary_freqs
from .paged import PagedPlan, paged_attn_fwd, paged_compress, paged_plan, paged_write
from .paged_q import paged_attn_q_fwd, paged_write_q

__version__ = "0.1.0"

__all__ = [
    "chunked_indexer_topk",
    "chunked_indexer_topk_quantized",
    "indexer_topk_q",
    "indexer_score",
    "indexer_score_topk",
    "sparse_attn",
    "sparse_attn_bwd",
    "sparse_attn_bwd_v2",
    "build_inverted_topk",
    "sparse_attn_fwd",
    "sparse_attn_fwd_kv2",
    "sparse_attn_kv2",
    "PagedPlan",
    "paged_plan",
    "paged_write",
    "paged_write_q",
    "paged_compress",
    "paged_attn_fwd",
    "paged_attn_q_fwd",
    "flash_hca_paged_forward",
    "rotary",
    "norm_rotary",
    "rotary_freqs",
    "flash_csa_forward",
    "build_csa_topk_idxs",
    "csa_topk_idxs",
    "flash_hca_forward",
    "build_hca_topk_idxs",
]
