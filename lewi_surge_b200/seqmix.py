"""Host-side mirror of the reference's sequence-mixing patches, backed by the sm_100a kernels.

`causal_conv1d(x, w)` is the causal depthwise 1-D convolution the reference rewrites as shift-adds
(`_fast_call`, modal/fast_conv.py:14-31): x [B,T,C] bf16, w [K,1,C] (the flax kernel layout) -> y [B,T,C].
Differentiable through `torch.autograd`; no fallback path.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import LewiError, check, ptr, stream


class _CausalConv1d(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, w):
    lib = _lib.load()
    if x.dim() != 3 or w.dim() != 3 or w.shape[1] != 1 or w.shape[2] != x.shape[2]:
      raise LewiError("causal_conv1d: x [B,T,C] and a depthwise kernel w [K,1,C] are required")
    if x.dtype != torch.bfloat16:
      raise LewiError("causal_conv1d takes bfloat16 activations")
    x = x.contiguous()
    wb = w.to(torch.bfloat16).contiguous()
    b, t, c = x.shape
    y = torch.empty_like(x)
    check(lib.lewi_causal_conv1d_fwd(stream(), ptr(x), ptr(wb), ptr(y), b, t, c, w.shape[0]), "lewi_causal_conv1d_fwd")
    ctx.save_for_backward(x, wb)
    ctx.w_dtype = w.dtype
    return y

  @staticmethod
  def backward(ctx, g):
    lib = _lib.load()
    x, wb = ctx.saved_tensors
    b, t, c = x.shape
    k = wb.shape[0]
    g = g.contiguous()
    dx = torch.empty_like(x)
    dw = torch.empty((k, 1, c), dtype=torch.float32, device=x.device)
    ws_bytes = int(lib.lewi_causal_conv1d_workspace_bytes(b, t, c, k))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
    check(lib.lewi_causal_conv1d_bwd(stream(), ptr(x), ptr(wb), ptr(g), ptr(dx), ptr(dw), _lib.F32, ptr(ws), ws_bytes, b, t,
                                     c, k), "lewi_causal_conv1d_bwd")
    return dx, dw.to(ctx.w_dtype)


def causal_conv1d(x, w):
  """y[b,t,c] = sum_j w[j,0,c] * x[b, t-(K-1)+j, c] (zero before the sequence starts).  Reference:
  `_fast_call`, modal/fast_conv.py:14-31."""
  return _CausalConv1d.apply(x, w)


class _ChunkGatedDeltaRule(torch.autograd.Function):
  """o, final state = chunked gated delta rule; the backward pass is `lewi_gdn_chunk_bwd`."""

  @staticmethod
  def forward(ctx, q, k, v, g, beta, h0):
    lib = _lib.load()
    b, s, h, kd = k.shape
    vd = v.shape[-1]
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    gf = g.to(torch.float32).contiguous()
    bb = beta.to(torch.bfloat16).contiguous()
    o = torch.empty((b, s, h, vd), dtype=torch.bfloat16, device=q.device)
    h0f = h0.to(torch.float32).contiguous() if h0 is not None else None
    hf = torch.empty((b, h, kd, vd), dtype=torch.float32, device=q.device)
    ws_bytes = int(lib.lewi_gdn_chunk_workspace_bytes(b, s, h, kd, vd))
    if ws_bytes < 0:
      check(ws_bytes, "lewi_gdn_chunk_workspace_bytes")
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    check(lib.lewi_gdn_chunk_fwd(stream(), ptr(q), ptr(k), ptr(v), ptr(gf), ptr(bb), ptr(h0f), ptr(o), ptr(hf), ptr(ws),
                                 ws_bytes, b, s, h, kd, vd), "lewi_gdn_chunk_fwd")
    ctx.save_for_backward(q, k, v, gf, bb, h0f, ws)
    ctx.set_materialize_grads(False)   # an output nobody differentiates arrives as None, not as a tensor of zeros
    ctx.in_dtypes = (g.dtype, beta.dtype, h0.dtype if h0 is not None else None)
    return o, hf

  @staticmethod
  def backward(ctx, d_o, d_hf):
    lib = _lib.load()
    q, k, v, gf, bb, h0f, ws = ctx.saved_tensors
    b, s, h, kd = k.shape
    vd = v.shape[-1]
    d_o = d_o.to(torch.bfloat16).contiguous() if d_o is not None else torch.zeros_like(v)
    d_hf = d_hf.to(torch.float32).contiguous() if d_hf is not None else None
    bws_bytes = int(lib.lewi_gdn_chunk_bwd_workspace_bytes(b, s, h, kd, vd))
    if bws_bytes < 0:
      check(bws_bytes, "lewi_gdn_chunk_bwd_workspace_bytes")
    bws = torch.empty(bws_bytes, dtype=torch.uint8, device=q.device)
    dq, dk, dv, db = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(bb)
    dg = torch.empty_like(gf)
    dh0 = torch.empty_like(h0f) if h0f is not None else None
    check(lib.lewi_gdn_chunk_bwd(stream(), ptr(q), ptr(k), ptr(v), ptr(gf), ptr(bb), ptr(h0f), ptr(d_o), ptr(d_hf), ptr(ws),
                                 ws.numel(), ptr(bws), bws_bytes, ptr(dq), ptr(dk), ptr(dv), ptr(dg), ptr(db), ptr(dh0), b,
                                 s, h, kd, vd), "lewi_gdn_chunk_bwd")
    g_dt, b_dt, h_dt = ctx.in_dtypes
    return dq, dk, dv, dg.to(g_dt), db.to(b_dt), (dh0.to(h_dt) if dh0 is not None else None)


def chunk_gated_delta_rule(query, key, value, g, beta, chunk_size=64, initial_state=None, final_state_dtype=torch.bfloat16):
  """The chunked gated delta rule with the signature of the reference's `fast_chunk_gated_delta_rule`
  (modal/gdn_fast.py:37): query, key [B,S,H,K], value [B,S,H,V] bf16, g [B,S,H] (log decay), beta [B,S,H]; returns
  (o [B,S,H,V] bf16, final state [B,H,K,V] bf16 or None when no initial state was given, as the reference does).
  `final_state_dtype=torch.float32` returns the final state as the kernel holds it, which is what `gated_delta_step` or a further piece of the
  sequence goes on from without a rounding.
  Differentiable through `torch.autograd` in q, k, v, g, beta and the initial state (head dimensions up to 128)."""
  if chunk_size != 64:
    raise LewiError("chunk_gated_delta_rule: the kernels work in chunks of 64 tokens")
  if query.dtype != torch.bfloat16 or key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
    raise LewiError("chunk_gated_delta_rule takes bfloat16 q, k, v")
  if final_state_dtype not in _GATES:
    raise LewiError("chunk_gated_delta_rule returns its final state as bfloat16 or float32")
  o, hf = _ChunkGatedDeltaRule.apply(query, key, value, g, beta, initial_state)
  return o, (hf.to(final_state_dtype) if initial_state is not None else None)


_GATES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


def _check_slots(what, b, n_states, slots):
  if slots is None:
    if n_states < b:
      raise LewiError(f"{what}: {b} rows and no slots, but {n_states} states")
  elif slots.shape != (b,):
    raise LewiError(f"{what}: slots [B] are required")


def causal_conv1d_step(x, w, state, slots=None):
  """One more input of the sequences of `causal_conv1d`: x [B,C] bf16, w [K,1,C], state [N,K-1,C] bf16 holds the K-1 inputs before this
  one, oldest first (zeros at the start of a sequence) and is moved on in place.  Row b has the state slots[b] (int32 or int64; none:
  state b).  A negative slot is an idle row: zeros out, no state touched; a slot past the pool, or an earlier row's, as well, with
  `LEWI_STATUS_BAD_INDEX` in `_lib.last_status()`.  Not differentiable (operands that require a gradient are
  refused while gradients are recorded); the values are `causal_conv1d`'s bit for bit."""
  lib = _lib.load()
  xs, ws, ss = x.shape, w.shape, state.shape
  if len(xs) != 2 or len(ws) != 3 or ws[1] != 1 or ws[2] != xs[1]:
    raise LewiError("causal_conv1d_step: x [B,C] and a depthwise kernel w [K,1,C] are required")
  if x.dtype is not torch.bfloat16 or state.dtype is not torch.bfloat16:
    raise LewiError("causal_conv1d_step takes bfloat16 activations and state")
  (b, c), k = xs, ws[0]
  if len(ss) != 3 or ss[1] != k - 1 or ss[2] != c:
    raise LewiError("causal_conv1d_step: state [N,K-1,C] is required")
  _check_slots("causal_conv1d_step", b, ss[0], slots)
  _lib.fits("causal_conv1d_step", b, ss[0], c, k)
  _lib.no_derivative("causal_conv1d_step", x, w, state)
  if _lib.elsewhere(x, w, state, slots):
    with torch.cuda.device(x.device):
      return causal_conv1d_step(x, w, state, slots)
  x, x_rows = _lib.rows_of(x, 16)
  if w.dtype is not torch.bfloat16 or not w.is_contiguous():
    w = w.detach().to(torch.bfloat16).contiguous()
  slots = _lib.index_table(slots, "slots")
  y = torch.empty_like(x, memory_format=torch.contiguous_format)
  if b > 0:
    check(lib.lewi_causal_conv1d_step(stream(x), x.data_ptr(), x_rows, ptr(w), ptr(state), ptr(slots), y.data_ptr(), b, ss[0], c, k),
          "lewi_causal_conv1d_step")
    _lib.written(state)
  return y


def gated_delta_step(query, key, value, g, beta, state, slots=None):
  """One more token of the sequences of `chunk_gated_delta_rule`, with the same arguments without their S: query, key [B,Hk,K],
  value [B,H,V] bf16, g (log decay), beta [B,H] (float32 or bf16) and the state [N,H,K,V] float32, which is moved on in place; returns
  o [B,H,V] bf16.  H is a multiple of Hk: value head h has the query and key of head h // (H // Hk).  Row b has the state slots[b]
  (int32 or int64; none: state b); idle and refused rows are those of `causal_conv1d_step`.  K up to 128, K and V multiples of 8.
  Rows of the batch may lie apart (views of one projection need no copy).  Not differentiable, as `causal_conv1d_step`.  Everything is float32 inside, where
  `chunk_gated_delta_rule` rounds some products to bf16 as the reference does, so the two agree to bf16's precision."""
  lib = _lib.load()
  if not query.dtype is key.dtype is value.dtype is torch.bfloat16 or state.dtype is not torch.float32:
    raise LewiError("gated_delta_step takes bfloat16 q, k, v and a float32 state")
  qs, vs, ss = query.shape, value.shape, state.shape
  if len(qs) != 3 or key.shape != qs or len(vs) != 3 or vs[0] != qs[0]:
    raise LewiError("gated_delta_step: query, key [B,Hk,K] and value [B,H,V] are required")
  (b, hk, kd), (_, h, vd) = qs, vs
  if len(ss) != 4 or ss[1] != h or ss[2] != kd or ss[3] != vd:
    raise LewiError("gated_delta_step: state [N,H,K,V] is required")
  if g.shape != vs[:2] or beta.shape != vs[:2]:
    raise LewiError("gated_delta_step: g and beta [B,H] are required")
  _check_slots("gated_delta_step", b, ss[0], slots)
  g_type, beta_type = _GATES.get(g.dtype), _GATES.get(beta.dtype)
  if g_type is None or beta_type is None:
    raise LewiError("gated_delta_step takes float32 or bfloat16 g and beta")
  _lib.fits("gated_delta_step", b, ss[0], hk, h, kd, vd)
  _lib.no_derivative("gated_delta_step", query, key, value, g, beta, state)
  if _lib.elsewhere(query, key, value, g, beta, state, slots):
    with torch.cuda.device(query.device):
      return gated_delta_step(query, key, value, g, beta, state, slots)
  (q, q_rows), (k, k_rows), (v, v_rows) = _lib.rows_of(query, 2), _lib.rows_of(key, 2), _lib.rows_of(value, 2)
  g, beta, slots = g.contiguous(), beta.contiguous(), _lib.index_table(slots, "slots")
  o = torch.empty_like(v, memory_format=torch.contiguous_format)
  if b > 0:
    check(lib.lewi_gdn_step(stream(q), q.data_ptr(), q_rows, k.data_ptr(), k_rows, v.data_ptr(), v_rows, g.data_ptr(), g_type, beta.data_ptr(),
                            beta_type, ptr(state), ptr(slots), o.data_ptr(), b, ss[0], hk, h, kd, vd), "lewi_gdn_step")
    _lib.written(state)
  return o
