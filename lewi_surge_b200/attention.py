"""Softmax attention of the decoder block's full-attention layers, beside the mixers of `seqmix`: `causal_attention` over whole
sequences for training and prompts, the paged key-value cache (`paged_cache_write`, `paged_attention`) for decoding.

Everything is bfloat16 with float32 scores, softmax and sums; no fallback path."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import LewiError, check, ptr, stream


def _check_cache(what, key_cache, value_cache, block_tables, lengths):
  """Pages, tokens per page, heads and head dimension of the caches, and the distance of their pages."""
  if not key_cache.dtype is value_cache.dtype is torch.bfloat16:
    raise LewiError(f"{what} takes bfloat16 caches")
  shape, tables = key_cache.shape, block_tables.shape
  if len(shape) != 4 or value_cache.shape != shape or shape[3] == 0:
    raise LewiError(f"{what}: caches [pages, page, Hkv, D] of one shape are required")
  pages, page, heads, d = shape
  page_stride = page * heads * d
  if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
    for t in (key_cache, value_cache):
      inside = all(n == 1 or step == packed for n, step, packed in zip(shape[1:], t.stride()[1:], (heads * d, d, 1)))
      if not inside or (pages > 1 and t.stride(0) != key_cache.stride(0)):
        raise LewiError(f"{what}: pages that are contiguous and as far apart in both caches are required")
    if pages > 1:
      page_stride = key_cache.stride(0)
  if len(tables) != 2 or lengths.shape != tables[:1]:
    raise LewiError(f"{what}: block_tables [B, max_pages] and lengths [B] are required")
  _lib.fits(what, page, heads, d, tables[0], tables[1])
  return pages, page, heads, d, page_stride


def paged_cache_write(key, value, key_cache, value_cache, block_tables, lengths, cu_seqlens=None):
  """Writes new tokens into their cells: key, value [T, Hkv, D] bf16 are the LAST tokens of their sequences, whose `lengths` [B] already
  count them.  Tokens cu_seqlens[b] .. cu_seqlens[b+1] belong to sequence b; without `cu_seqlens` every sequence has one (T = B), and one
  of length 0 is idle.  Caches [pages, page, Hkv, D] bf16 (pages may lie apart: views of one tensor that interleaves both);
  sequence b's tokens lie in the pages block_tables[b] (int32 or int64) names.  Tokens of no sequence are left out.  A token that lies
  outside its sequence's table or on a page that does not exist is left out with `LEWI_STATUS_BAD_INDEX` in `_lib.last_status()`.
  Two tokens written to one cell (a page named twice) leave either of them, piece by piece.  Not differentiable, as `paged_attention`."""
  lib = _lib.load()
  pages, page, heads, d, page_stride = _check_cache("paged_cache_write", key_cache, value_cache, block_tables, lengths)
  new = key.shape
  if not key.dtype is value.dtype is torch.bfloat16 or len(new) != 3 or new[1] != heads or new[2] != d or value.shape != new:
    raise LewiError("paged_cache_write: key, value [T, Hkv, D] bfloat16, as wide as the caches, are required")
  t, (b, max_pages) = new[0], block_tables.shape
  _lib.fits("paged_cache_write", t, b)
  if cu_seqlens is not None and cu_seqlens.shape != (b + 1,):
    raise LewiError("paged_cache_write: cu_seqlens [B + 1] is required")
  if cu_seqlens is None and t != b:
    raise LewiError("paged_cache_write: without cu_seqlens there is one token per sequence")
  _lib.no_derivative("paged_cache_write", key, value, key_cache, value_cache)
  if t == 0 or b == 0:
    return
  if _lib.elsewhere(key_cache, key, value, value_cache, block_tables, lengths, cu_seqlens):
    with torch.cuda.device(key_cache.device):
      return paged_cache_write(key, value, key_cache, value_cache, block_tables, lengths, cu_seqlens)
  (k, ks), (v, vs) = _lib.rows_of(key, 16), _lib.rows_of(value, 16)
  tables, lens = _lib.index_table(block_tables, "block_tables"), _lib.index_table(lengths, "lengths")
  cu = _lib.index_table(cu_seqlens, "cu_seqlens")
  check(lib.lewi_paged_cache_write(stream(k), k.data_ptr(), ks, v.data_ptr(), vs, key_cache.data_ptr(), value_cache.data_ptr(), page_stride,
                                   tables.data_ptr(), lens.data_ptr(), ptr(cu), t, b, heads, d, pages, page, max_pages), "lewi_paged_cache_write")
  _lib.written(key_cache, value_cache)


def paged_attention(query, key_cache, value_cache, block_tables, lengths, scale=None):
  """Attention of one new token per sequence over the sequence's cells, its own among them (write it first): query [B, Hq, D] bf16 ->
  [B, Hq, D] bf16, head h with the keys of head h // (Hq // Hkv); zeros where lengths[b] is 0.  Caches and tables as in
  `paged_cache_write`; D up to 256, a multiple of 8.  `scale` defaults to D ** -0.5.  Not differentiable: operands that
  require a gradient are refused while gradients are recorded.  Lengths and tables are read on the device, so a
  captured call follows them.  Cells past a sequence's length, whatever they hold, have no part in it; pages that do not exist
  and what a length has past its table are left out with `LEWI_STATUS_BAD_INDEX` in `_lib.last_status()`."""
  lib = _lib.load()
  pages, page, heads, d, page_stride = _check_cache("paged_attention", key_cache, value_cache, block_tables, lengths)
  shape, (b, max_pages) = query.shape, block_tables.shape
  if query.dtype is not torch.bfloat16 or len(shape) != 3 or shape[2] != d or heads == 0 or shape[1] % heads or shape[0] != b:
    raise LewiError("paged_attention: query [B, Hq, D] bfloat16 with Hq a multiple of the caches' heads is required")
  _lib.no_derivative("paged_attention", query, key_cache, value_cache)
  hq = shape[1]
  _lib.fits("paged_attention", hq, b)
  if _lib.elsewhere(query, key_cache, value_cache, block_tables, lengths):
    with torch.cuda.device(query.device):
      return paged_attention(query, key_cache, value_cache, block_tables, lengths, scale)
  q, qs = _lib.rows_of(query, 4)
  o = torch.empty_like(q, memory_format=torch.contiguous_format)
  if b == 0 or hq == 0:
    return o
  tables, lens = _lib.index_table(block_tables, "block_tables"), _lib.index_table(lengths, "lengths")
  ws_bytes = lib.lewi_paged_attention_workspace_bytes(d)
  if ws_bytes < 0:
    check(ws_bytes, "lewi_paged_attention_workspace_bytes")
  ws = q.new_empty(ws_bytes // 2)
  check(lib.lewi_paged_attention(stream(q), q.data_ptr(), qs, key_cache.data_ptr(), value_cache.data_ptr(), page_stride, tables.data_ptr(),
                                 lens.data_ptr(), o.data_ptr(), ws.data_ptr(), ws_bytes, b, hq, heads, d, pages, page, max_pages,
                                 d ** -0.5 if scale is None else float(scale)), "lewi_paged_attention")
  return o


_CHAIN_ROWS = 32768   # rows of a sequence from which on the forward pass keeps sums in `o_rest` (more go into no accumulator)


def _attention_fwd(q, k, v, cu, n_seqs, scale, o_rest=None, lse=None):
  """Output, the operands as the kernels read them and the distances of their rows; `o_rest` like the output and `lse` [Hq, T] receive
  what the backward pass needs."""
  (q, q_rows), (k, k_rows), (v, v_rows) = _lib.rows_of(q, 16), _lib.rows_of(k, 16), _lib.rows_of(v, 16)
  cu = _lib.index_table(cu, "cu_seqlens")
  t, hq, d = q.shape
  o = torch.empty_like(q, memory_format=torch.contiguous_format)
  if o_rest is None and t > _CHAIN_ROWS:
    o_rest = torch.empty_like(o)
  check(_lib.load().lewi_causal_attention_fwd(stream(q), q.data_ptr(), q_rows, k.data_ptr(), k_rows, v.data_ptr(), v_rows, ptr(cu), n_seqs,
                                              o.data_ptr(), ptr(o_rest), ptr(lse), t, hq, k.shape[1], d, scale), "lewi_causal_attention_fwd")
  return o, q, k, v, cu, (q_rows, k_rows, v_rows)


class _CausalAttention(torch.autograd.Function):

  @staticmethod
  def forward(ctx, q, k, v, cu, n_seqs, scale):
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device)
    o_rest = torch.empty_like(q, memory_format=torch.contiguous_format)
    o, q, k, v, cu, rows = _attention_fwd(q, k, v, cu, n_seqs, scale, o_rest, lse)
    ctx.save_for_backward(q, k, v, o, o_rest, lse, cu)
    ctx.call = n_seqs, scale, rows
    return o

  @staticmethod
  def backward(ctx, g):
    if torch.is_grad_enabled():   # (create_graph: what these kernels do would be missing from it)
      raise LewiError("causal_attention is differentiable once")
    lib = _lib.load()
    q, k, v, o, o_rest, lse, cu = ctx.saved_tensors
    n_seqs, scale, (q_rows, k_rows, v_rows) = ctx.call
    (t, hq, d), hkv = q.shape, k.shape[1]
    g, _ = _lib.rows_of(g.contiguous(), 16)
    need_q, need_k, need_v = ctx.needs_input_grad[:3]
    dq = o.new_empty((t, hq, d)) if need_q else None
    dk, dv = (o.new_empty((t, hkv, d)), o.new_empty((t, hkv, d))) if need_k or need_v else (None, None)
    ws_bytes = lib.lewi_causal_attention_bwd_workspace_bytes(t, n_seqs, hq, hkv, d)
    ws = lse.new_empty((ws_bytes + 3) // 4)
    check(lib.lewi_causal_attention_bwd(stream(), q.data_ptr(), q_rows, k.data_ptr(), k_rows, v.data_ptr(), v_rows, o.data_ptr(),
                                        o_rest.data_ptr(), lse.data_ptr(), g.data_ptr(), ptr(cu), n_seqs, ptr(dq), ptr(dk), ptr(dv),
                                        ws.data_ptr(), ws_bytes, t, hq, hkv, d, scale),
          "lewi_causal_attention_bwd")
    return dq, dk, dv, None, None, None


def causal_attention(query, key, value, cu_seqlens=None, scale=None):
  """softmax(scale q k^T) v over the rows of a sequence up to the query's own.  Packed: query [T, Hq, D], key, value [T, Hkv, D] bf16, sequence s
  the rows cu_seqlens[s] .. cu_seqlens[s+1] (int32 or int64 [N + 1], ascending, empty ones among them; none: one sequence), or sequences of one
  length: query [B, S, Hq, D], key, value [B, S, Hkv, D].  Head h has the keys of head h // (Hq // Hkv); D up to 128, a multiple of 8;
  `scale` > 0 defaults to D ** -0.5.  Returns bf16 of the query's shape; differentiable through `torch.autograd`, once and
  in reverse mode, in query, key and value.
  Rows of no sequence give zeros and get zero gradients, whatever they hold.  Bounds that leave the rows are cut to them; where bounds fall, no
  sequence is worked on and the results are undefined; either way `LEWI_STATUS_BAD_INDEX` in `_lib.last_status()`.  Rows may lie apart (views of one projection need no copy).

  Outputs with and without gradients wanted may differ by a rounding in the first 128 rows of a sequence, whose p are kept to 2^-16 for the former.

  A value of v that is not finite reaches back to the start of its 128 rows of the sequence (as those of q, k and the upstream gradient do in the
  gradients), never into another sequence."""
  if not query.dtype is key.dtype is value.dtype is torch.bfloat16:
    raise LewiError("causal_attention takes bfloat16 q, k, v")
  shape, other = query.shape, key.shape
  n = len(shape)
  if n not in (3, 4) or len(other) != n or value.shape != other or shape[:-2] != other[:-2] or shape[-1] != other[-1] or other[-2] == 0 or \
      shape[-2] % other[-2]:
    raise LewiError("causal_attention: query [T, Hq, D] and key, value [T, Hkv, D], or all three [B, S, ..], Hq a multiple of Hkv, are required")
  n_seqs = 1 if n == 3 else shape[0]
  _lib.fits("causal_attention", shape[0] * (shape[1] if n == 4 else 1), shape[-2], shape[-1])
  if cu_seqlens is not None:
    if n == 4 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
      raise LewiError("causal_attention: cu_seqlens [N + 1] belongs to packed rows [T, H, D]")
    n_seqs = cu_seqlens.shape[0] - 1
    _lib.fits("causal_attention", n_seqs)
  scale = max(shape[-1], 1) ** -0.5 if scale is None else float(scale)
  if not 0 < scale < 2e38:
    raise LewiError("causal_attention: scale must be positive, and float32 must hold it")
  if torch.autograd.forward_ad._current_level >= 0 and _lib.has_tangent(query, key, value):
    raise LewiError("causal_attention has no forward-mode derivative")
  if query.numel() == 0:
    return query + 0 * (key.sum() + value.sum())   # (nothing, with gradients of zero)
  if _lib.elsewhere(query, key, value, cu_seqlens):
    with torch.cuda.device(query.device):
      return causal_attention(query, key, value, cu_seqlens, scale)
  if n == 4:
    query, key, value = (x.reshape(-1, *x.shape[2:]) for x in (query, key, value))
  if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
    o = _CausalAttention.apply(query, key, value, cu_seqlens, n_seqs, scale)
  else:
    o = _attention_fwd(query, key, value, cu_seqlens, n_seqs, scale)[0]
  return o if n == 3 else o.view(shape)
