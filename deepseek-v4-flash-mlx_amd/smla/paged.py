"""The paged latent cache: a pool of pages that many sequences of unlike lengths share.

The reference keeps one contiguous buffer a sequence and clones it whole
(``oracle/v4_fast.py:93-96,150-159``); a server that batches sequences keeps their rows in pages
instead.  Row j of sequence b is row j % P of page ``table[b, j // P]`` of ``pages`` [n_pages, P, D]
(bf16, or e4m3 codes with ``page_scales`` [n_pages, P, D/64], whose products with the codes the attention takes as bf16:
exactly where they are powers of two, as the append makes them).  A step is

* ``update_pages``   slots forked, freed and grown (new ``table``, ``lens``, ``refs``);
* ``paged_append``   the new tokens' queries normed and rotated, their rows written to the pages;
* ``paged_attn``     the tokens' attention over their sequences' rows;

and between steps ``compact_pages`` moves the live pages to the pool's start.  Lengths, tables and
counts are int32 tensors on the GPU that the host never reads, so a step can be captured once and replayed.
All calls are stream-ordered.
"""
import torch

from . import _lib, ops


def paged_attn(q, pages, table, lens, cu, scale, attn_sink=None, window=0, first=0, dv=512, page_scales=None, out=None,
               granted=None):
    """Attention of a ragged batch's newest tokens: q [T, H, D] bf16 (D 512 or 576), of sequence b the
    tokens cu[b] .. cu[b+1]-1, the last rows of its lens[b]; table [B, cols], lens [B], cu [B+1] int32.
    A token at position p attends rows j <= p, with window > 0 those with j > p - window or
    j < first; ``attn_sink`` [H] adds to the denominator as in ``sparse_attn``; a token that sees no
    row gives 0.  Returns [T, H, dv] bf16: ``out`` when given (apart from q; tokens of no sequence are
    left as they were), else a new tensor (0 there).  ``granted`` [B] int32 (``update_pages``): the tokens of a sequence
    where it is 0 are tokens of no sequence.  One token a sequence, a prompt's chunk and any mix of them are the same
    call."""
    fill = out is None
    if fill:
        if q.dim() != 3:
            raise ValueError("expected q [T,H,D]")
        out = torch.empty(q.shape[0], q.shape[1], dv, dtype=torch.bfloat16, device=q.device)
    ops.paged_attn_op_(q, pages, page_scales, table, lens, cu, attn_sink, float(scale), int(window), int(first), fill, out,
                       granted)
    return out


def paged_append(q, kv, pages, table, lens, cu, cos_t, sin_t, kv_norm=None, q_norm=None, norm_dims=None,
                 page_scales=None, fp8_sim=False, eps=1e-6, q_out=None, granted=None):
    """The new tokens' queries and rows from their projections, in one launch: q [T, H, D] (None: rows
    only) and kv [T, D], fp32 or bf16 (row-strided slices pass as they are).  ``q_norm`` / ``kv_norm``: None or False no
    norm, True the weightless one, a tensor [norm_dims] its weights; norm_dims (default: min(D, 512)) leading channels are
    RMS-normed, then the last 2 * cos_t.shape[1] channels rotated to the token's position (``norm_rope.rope_tables``).
    The rows go to their pages: bf16 (``fp8_sim``: the channels before the rotated ones fp8
    round-tripped first) or, with fp8 pages, e4m3 codes and ``page_scales``.  Returns the queries [T, H, D] bf16
    (``q_out`` when given: tokens of no sequence or at positions past the rotation tables are left as
    they were; else 0 there; apart from q and kv, or q itself where that is dense bf16), None without q.  ``granted`` [B] int32 (``update_pages``): the tokens of a sequence
    where it is 0 are tokens of no sequence; without it they are written over the refused slot's last rows."""
    fill = q is not None and q_out is None
    if fill:
        if q.dim() != 3:
            raise ValueError("expected q [T,H,D]")
        q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    if q is None and q_out is not None:
        raise ValueError("q_out without q")
    flags = _lib.PAGED_FILL if fill else 0
    q_weights = kv_weights = None
    if isinstance(q_norm, torch.Tensor):
        q_weights, flags = q_norm, flags | _lib.PAGED_NORM_Q
    elif q_norm:
        flags |= _lib.PAGED_NORM_Q
    if isinstance(kv_norm, torch.Tensor):
        kv_weights, flags = kv_norm, flags | _lib.PAGED_NORM_KV
    elif kv_norm:
        flags |= _lib.PAGED_NORM_KV
    if norm_dims is None:
        norm_dims = min(kv.shape[-1], 512)
    ops.paged_append_op_(q, kv, pages, page_scales, table, lens, cu, cos_t, sin_t, q_weights, kv_weights, int(norm_dims),
                         bool(fp8_sim), float(eps), flags, q_out, granted)
    return q_out


def update_pages(pages, table, lens, refs, parent, grow, page_scales=None):
    """Every slot's next state at once: slot s becomes a copy of slot parent[s] as before the call (s: itself, -1: an
    empty slot) and grows by grow[s] rows, or gives its last -grow[s] rows back.  Whole pages are shared, a copied
    slot's partly filled last page is copied to a fresh one, fresh pages are the free ones (refs 0) in ascending order.
    pages [n_pages, P, D] or [layers, n_pages, P, D] (layers under one table), table [S, M], lens / parent / grow [S],
    refs [n_pages] int32.  Returns new (table, lens, refs, granted), the state of the next call (lengths change here
    only); granted[s] = 0 marks a slot left as it was (arguments out of range, more than M pages, or not enough free
    pages for slots 0 .. s): it has no rows for its new tokens, so pass granted on to ``paged_append`` and
    ``paged_attn``.  Freeing is parent -1, grow 0; beam reordering any map; a new sequence of n rows parent -1, grow n;
    a step after rejected drafts grow = new tokens - rejected ones (given back by a call of their own, grow < 0, where
    another slot was made a copy of this one since they were written, in the same call too)."""
    return ops.update_pages_op(pages, page_scales, table, lens, refs, parent, grow)


def compact_pages(pages, table, refs, page_scales=None):
    """The live pages (refs > 0) moved together: the i-th live page past their number goes to the i-th free id
    below it, in place and in every layer.  Returns new (table, refs, live): entries follow their pages (-1
    where an entry names no live page), live [1] is the number of pages in use."""
    return ops.compact_pages_op(pages, page_scales, table, refs)
