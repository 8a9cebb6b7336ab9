"""Softmax attention of the decoder block's full-attention layers, beside the mixers of `seqmix`: the paged key-value cache
(`paged_cache_write`, `paged_attention`) for decoding.

Everything is bfloat16 with float32 scores, softmax and sums; no fallback path."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import LewiError, check, ptr, stream


def _check_cache(what, key_cache, value_cache, block_tables, lengths):
  if key_cache.dtype != torch.bfloat16 or value_cache.dtype != torch.bfloat16:
    raise LewiError(f"{what} takes bfloat16 caches")
  if key_cache.dim() != 4 or value_cache.shape != key_cache.shape:
    raise LewiError(f"{what}: caches [pages, page, Hkv, D] of one shape are required")
  _, page, heads, d = key_cache.shape
  for t in (key_cache, value_cache):
    if t.stride()[1:] != (heads * d, d, 1) or (t.shape[0] > 1 and t.stride(0) != key_cache.stride(0)):
      raise LewiError(f"{what}: pages that are contiguous and as far apart in both caches are required")
  if block_tables.dim() != 2 or lengths.shape != (block_tables.shape[0],):
    raise LewiError(f"{what}: block_tables [B, max_pages] and lengths [B] are required")
  page_stride = key_cache.stride(0) if key_cache.shape[0] > 1 else page * heads * d
  return page_stride, page, heads, d


def paged_cache_write(key, value, key_cache, value_cache, block_tables, lengths, cu_seqlens=None):
  """Writes new tokens into their cells: key, value [T, Hkv, D] bf16 are the LAST tokens of their sequences, whose `lengths` [B] already
  count them.  Tokens cu_seqlens[b] .. cu_seqlens[b+1] belong to sequence b; without `cu_seqlens` every sequence has one (T = B), and one
  of length 0 is idle.  Caches [pages, page, Hkv, D] bf16 (pages may lie apart: views of one tensor that interleaves both);
  sequence b's tokens lie in the pages block_tables[b] (int32 or int64) names.  Tokens of no sequence are left out.  A token that lies
  outside its sequence's table or on a page that does not exist is left out with `LEWI_STATUS_BAD_INDEX` in `_lib.last_status()`.
  Two tokens written to one cell (a page named twice) leave either of them, piece by piece."""
  lib = _lib.load()
  page_stride, page, heads, d = _check_cache("paged_cache_write", key_cache, value_cache, block_tables, lengths)
  if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16 or key.dim() != 3 or key.shape[1:] != (heads, d) or value.shape != key.shape:
    raise LewiError("paged_cache_write: key, value [T, Hkv, D] bfloat16, as wide as the caches, are required")
  t, b = key.shape[0], block_tables.shape[0]
  if cu_seqlens is not None and cu_seqlens.shape != (b + 1,):
    raise LewiError("paged_cache_write: cu_seqlens [B + 1] is required")
  if cu_seqlens is None and t != b:
    raise LewiError("paged_cache_write: without cu_seqlens there is one token per sequence")
  if t == 0 or b == 0:
    return
  with torch.no_grad(), _lib.one_device(key, value, key_cache, value_cache, block_tables, lengths, cu_seqlens):
    (k, ks), (v, vs) = _lib.rows_of(key, 16), _lib.rows_of(value, 16)
    tables, lens, cu = (_lib.index_table(x, n) for x, n in ((block_tables, "block_tables"), (lengths, "lengths"), (cu_seqlens, "cu_seqlens")))
    check(lib.lewi_paged_cache_write(stream(), k.data_ptr(), ks, v.data_ptr(), vs, key_cache.data_ptr(), value_cache.data_ptr(), page_stride,
                                     ptr(tables), ptr(lens), ptr(cu), t, b, heads, d, key_cache.shape[0], page, tables.shape[1]),
          "lewi_paged_cache_write")


def paged_attention(query, key_cache, value_cache, block_tables, lengths, scale=None):
  """Attention of one new token per sequence over the sequence's cells, its own among them (write it first): query [B, Hq, D] bf16 ->
  [B, Hq, D] bf16, head h with the keys of head h // (Hq // Hkv); zeros where lengths[b] is 0.  Caches and tables as in
  `paged_cache_write`; D up to 256, a multiple of 8.  `scale` defaults to D ** -0.5.  Lengths and tables are read on the device, so a
  captured call follows them.  Cells past a sequence's length, whatever they hold, have no part in it; pages that do not exist
  and what a length has past its table are left out with `LEWI_STATUS_BAD_INDEX` in `_lib.last_status()`."""
  lib = _lib.load()
  page_stride, page, heads, d = _check_cache("paged_attention", key_cache, value_cache, block_tables, lengths)
  if query.dtype != torch.bfloat16 or query.dim() != 3 or query.shape[2] != d or query.shape[1] % heads or query.shape[0] != block_tables.shape[0]:
    raise LewiError("paged_attention: query [B, Hq, D] bfloat16 with Hq a multiple of the caches' heads is required")
  b, hq = query.shape[:2]
  with torch.no_grad(), _lib.one_device(query, key_cache, value_cache, block_tables, lengths):
    q, qs = _lib.rows_of(query, 4)
    o = torch.empty((b, hq, d), dtype=torch.bfloat16, device=q.device)
    if b == 0 or hq == 0:
      return o
    tables, lens = _lib.index_table(block_tables, "block_tables"), _lib.index_table(lengths, "lengths")
    ws_bytes = int(lib.lewi_paged_attention_workspace_bytes(d))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    check(lib.lewi_paged_attention(stream(), q.data_ptr(), qs, key_cache.data_ptr(), value_cache.data_ptr(), page_stride, ptr(tables), ptr(lens),
                                   ptr(o), ptr(ws), ws_bytes, b, hq, heads, d, key_cache.shape[0], page, tables.shape[1],
                                   d ** -0.5 if scale is None else float(scale)), "lewi_paged_attention")
  return o
