"""Attention of new tokens over a paged KV cache (``qik.paged_kv``), next to the block-causal
attention over a contiguous slab of ``qik.triton_attention``.

One call serves a batch of sequences that each bring one token (decoding), a few (drafts),
a chunk or a whole prompt; query heads may share key heads; rows see the cache causally, or
all of it, or the last ``window`` keys and the first ``sinks``.  The kernels
(``csrc/qik_paged_attn.cu``) read the lengths on the device, so a captured graph follows them.
"""
from __future__ import annotations

import torch

from . import _calls


def paged_attention(
    q: torch.Tensor,             # [T, HQ, D] new tokens of all sequences, one after another
    k_pages: torch.Tensor,       # [pages, HK, page, D]
    v_pages: torch.Tensor,
    page_table: torch.Tensor,    # [B, W] int32
    seq_lens: torch.Tensor,      # [B] int32: tokens in the cache, the new ones among them
    query_starts: torch.Tensor,  # [B + 1] int32: sequence i's rows of q
    max_new: int,                # most new tokens of a sequence
    max_kv: int | None = None,   # most tokens of a sequence (None: what the page table can hold)
    sm_scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    sinks: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """softmax(q . k * sm_scale) . v of each new token over its sequence's keys, [T, HQ, D].

    The new tokens are the last of their sequence, already stored.  Row j of n in a sequence of
    ``kv`` tokens sees the keys t <= kv - n + j (``causal``) or all kv; with ``window`` (causal
    only) those with t > kv - n + j - window or t < ``sinks``.  A row that sees nothing is 0.
    Places that a row does not see may hold anything, NaN included (a row that others of its
    tile see infinities beside is formed a second time, which takes longer).  ``sm_scale`` is
    D ** -0.5 by default.  Sums are fp32; the probabilities are rounded to q's type before the
    product with v, as the matrix instructions take them.

    ``out`` ([T, HQ, D], unit column stride) receives the result and may share no memory with q
    or the pages: other heads or tokens of q's allocation are fine, a view that cannot be told
    apart from what is read is refused.  Rows behind query_starts[B] are not written.

    ``query_starts`` ascend; no sequence may bring more than ``max_new`` tokens; ``max_kv`` only
    chooses launch shapes.  Lengths, starts and page numbers outside their tensors are skipped
    and set ``STATUS_BAD_INDEX`` (``qik._lib.device_status``)."""
    return _calls.paged_attention(q, k_pages, v_pages, page_table, seq_lens, query_starts, max_new, max_kv, sm_scale,
                                  causal, window, sinks, out)
