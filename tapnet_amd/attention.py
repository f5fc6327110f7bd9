"""Operators of a learned readout of a clip's feature grids: layer normalisation, rotary positions of several axes and
cross attention of point queries to feature tokens, with their gradients.

They stand beside the fixed readout of the TAPIR path (the cost volume and its soft arg max,
tapnet/models/tapir_model.py:399-471): ``TAPIR.get_feature_grids`` gives the tokens ``[batch, frames * h * w, channels]``
that points attend to, their (t, y, x) coordinates are the positions.  Everything runs in hand-written gfx950 kernels
through the C ABI (``include/tapir_hip.h``); there is no CPU fallback.  Element types are the engine's two, float32 and
bfloat16; sums, statistics and the parameters of a norm are float32 in both.

Calls are enqueued on the current stream of the tensors' device, whatever the current device is; nothing synchronises.
Scratch memory comes from torch's allocator, so calls on several streams and captured graphs do not share any.  A graph
may capture them once a call of the same element type has been made on the device (it loads the library).  No kernel uses
atomics: the same call gives the same bits.
"""
from __future__ import annotations

import ctypes
import math
import threading
from typing import Optional, Sequence, Union

import torch

from tapnet_amd import _ffi

_DTYPES = {torch.float32: _ffi.TAPIR_F32, torch.bfloat16: _ffi.TAPIR_BF16}
_lock = threading.Lock()
_contexts = {}


def _context(device: torch.device, dtype: torch.dtype):
  """The context of a device and element type.  It holds no weights and no workspaces, only the last error's text."""
  key = (device.index, dtype)
  ctx = _contexts.get(key)
  if ctx is None:
    if torch.cuda.is_current_stream_capturing():
      raise RuntimeError('call the operator once before capturing it into a graph (the first call loads the library)')
    lib = _ffi.load_library()
    cfg = _ffi.TapirCfg(1, 4, 12, 0, 20.0, 256, 256, _DTYPES[dtype])
    ctx = ctypes.c_void_p()
    _ffi.check(lib, None, lib.tapir_create(ctypes.byref(ctx), ctypes.byref(cfg), device.index), 'tapir_create')
    _contexts[key] = ctx
  return ctx


def _call(like: torch.Tensor, name: str, *args, on_stream: bool = True):
  """One C call in the context of `like`'s device and type.  Contexts are not thread-safe: calls take turns."""
  with torch.cuda.device(like.device), _lock:
    ctx = _context(like.device, like.dtype)
    lib = _ffi.load_library()
    if on_stream:
      args += (torch.cuda.current_stream().cuda_stream,)
    _ffi.check(lib, ctx, getattr(lib, name)(ctx, *args), name)


def _check_tensor(name: str, t, ndim: Optional[int] = None, like: Optional[torch.Tensor] = None):
  if not isinstance(t, torch.Tensor):
    raise TypeError(f'{name} has to be a torch tensor')
  if like is None:
    if t.dtype not in _DTYPES:
      raise ValueError(f'{name} has to be float32 or bfloat16, not {t.dtype}')
    if t.device.type != 'cuda':
      raise ValueError(f'{name} has to be on the GPU: tapnet_amd has no CPU fallback')
  else:
    if t.device != like.device:
      raise ValueError(f'{name} is on {t.device}, the input on {like.device}')
  if ndim is not None and t.ndim != ndim:
    raise ValueError(f'{name} has to have {ndim} axes, not {t.ndim}')


def _aligned(t: torch.Tensor) -> torch.Tensor:
  """`t` itself where its rows (last axis) are dense and start at multiples of 16 bytes, else a dense copy."""
  epc = 16 // t.element_size()
  if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % epc == 0 for s in t.stride()[:-1]):
    return t
  t = t.contiguous()
  return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
  return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t: Optional[torch.Tensor]):
  return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------------------ layer norm
def _rows(x: torch.Tensor):
  """x as [rows, channels] with dense channels and one row stride (a view where the strides allow it), and that stride."""
  channels = x.shape[-1]
  try:
    flat = x.view(-1, channels)
  except RuntimeError:
    flat = x.contiguous().view(-1, channels)
  if flat.stride(-1) != 1 and channels > 1:
    flat = flat.contiguous()
  return flat, flat.stride(0)


class _LayerNorm(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, weight, bias, eps, train):
    flat, stride = _rows(x)
    rows, channels = flat.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean, rstd = (torch.empty((2, rows), dtype=torch.float32, device=x.device) if train else (None, None))
    _call(x, 'tapir_layer_norm', flat.data_ptr(), stride, _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(mean), _ptr(rstd),
          rows, channels, eps)
    if train:
      ctx.save_for_backward(x, weight, mean, rstd)
    return y

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, dy):
    x, weight, mean, rstd = ctx.saved_tensors
    flat, stride = _rows(x)
    dflat, dstride = _rows(dy)
    rows, channels = flat.shape
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dgamma = torch.empty(channels, dtype=torch.float32, device=x.device) if ctx.needs_input_grad[1] else None
    dbeta = torch.empty(channels, dtype=torch.float32, device=x.device) if ctx.needs_input_grad[2] else None
    work = None
    if dgamma is not None or dbeta is not None:
      nbytes = ctypes.c_uint64()
      _call(x, 'tapir_layer_norm_workspace', rows, channels, ctypes.byref(nbytes), on_stream=False)
      work = _workspace(nbytes.value, x.device)
    _call(x, 'tapir_layer_norm_backward', flat.data_ptr(), stride, dflat.data_ptr(), dstride, _ptr(weight),
          mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), _ptr(dgamma), _ptr(dbeta), rows, channels, _ptr(work),
          work.numel() if work is not None else 0)
    return dx, dgamma, dbeta, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
  """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, as the norms of the PIPs mixer (scale only,
  tapnet/models/tapir_model.py:70-77) and of ExtraConvs (:176) have it, for any shape, and with gradients.

  x: float32 or bfloat16 ``[..., channels]`` of any strides.  weight, bias: float32 ``[channels]`` or None.  Statistics
  and sums are float32; the result has x's type.  Gradients of x (its type), weight and bias (float32)."""
  _check_tensor('x', x)
  if x.ndim < 1 or x.shape[-1] < 1:
    raise ValueError('x has to have a last axis of at least one channel')
  for name, p in (('weight', weight), ('bias', bias)):
    if p is None:
      continue
    _check_tensor(name, p, 1, like=x)
    if p.dtype != torch.float32 or p.shape[0] != x.shape[-1]:
      raise ValueError(f'{name} has to be float32 [{x.shape[-1]}], not {p.dtype} {list(p.shape)}')
  if not (eps >= 0 and math.isfinite(eps)):
    raise ValueError(f'eps has to be finite and not negative, not {eps}')
  if weight is not None:
    weight = weight.contiguous()
  if bias is not None:
    bias = bias.contiguous()
  train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias))
  return _LayerNorm.apply(x, weight, bias, float(eps), train)


# ------------------------------------------------------------------------------------------------ rotary positions
def _rotate(x, positions, sections, bases, interleaved, inverse):
  if x.stride(-1) != 1 and x.shape[-1] > 1:
    x = x.contiguous()
  batch, tokens, heads, dim = x.shape
  y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
  axes = len(sections)
  args = _ffi.TapirRotaryArgs(batch, tokens, heads, dim, axes, int(interleaved), int(inverse))
  args.section[:axes], args.base[:axes] = sections, bases
  args.x, args.x_stride[:], args.y = x.data_ptr(), x.stride()[:3], y.data_ptr()
  args.positions = positions.data_ptr()
  args.positions_stride = tokens * axes if positions.ndim == 3 and positions.shape[0] > 1 else 0
  _call(x, 'tapir_rotary_positions', ctypes.byref(args))
  return y


class _Rotary(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, positions, sections, bases, interleaved):
    ctx.save_for_backward(positions)
    ctx.how = (sections, bases, interleaved)
    return _rotate(x, positions, *ctx.how, False)

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, dy):
    return _rotate(dy, ctx.saved_tensors[0], *ctx.how, True), None, None, None, None


def rotary_positions(x: torch.Tensor, positions: torch.Tensor, sections: Optional[Sequence[int]] = None,
                     base: Union[float, Sequence[float]] = 10000.0, interleaved: bool = False) -> torch.Tensor:
  """Rotary positions of several axes -- (t, y, x) of a video token or a point between cells -- on queries or keys.

  x: float32 or bfloat16 ``[batch, tokens, heads, dim]`` of any strides, dim at most 256.  positions: float32
  ``[batch, tokens, axes]``, or ``[tokens, axes]`` for all clips alike; 1 to 4 axes, any real numbers (frames, pixels;
  angles are formed in 64 bits, so far positions keep their accuracy).  sections: even channel counts, one per axis, the
  first channels of a head for the first axis and so on; channels behind the last section pass through.  Default: the
  head's pairs in equal shares, what is left over a pair each to the first axes.  Pair i of a section of width w turns by
  ``position * base ** (-2 i / w)`` (base: one number, or one per axis); its two channels are i and i + w / 2 of the section,
  or neighbours with ``interleaved``.  The gradient goes to x; positions that require one are refused."""
  _check_tensor('x', x, 4)
  _check_tensor('positions', positions, like=x)
  batch, tokens, _, dim = x.shape
  if positions.dtype != torch.float32:
    raise ValueError(f'positions have to be float32, not {positions.dtype}')
  if positions.ndim not in (2, 3) or positions.shape[-2] != tokens or (
      positions.ndim == 3 and positions.shape[0] not in (1, batch)):
    raise ValueError(f'positions have to be [{batch}, {tokens}, axes] or [{tokens}, axes], not {list(positions.shape)}')
  if positions.requires_grad:
    raise ValueError('positions have no gradient: detach them')
  axes = positions.shape[-1]
  if not 1 <= axes <= 4:
    raise ValueError(f'1 to 4 axes of positions, not {axes}')
  if sections is None:
    pairs = dim // 2
    sections = [2 * (pairs // axes + (a < pairs % axes)) for a in range(axes)]
  sections = [int(s) for s in sections]
  if len(sections) != axes or any(s < 0 or s % 2 for s in sections) or sum(sections) > dim:
    raise ValueError(f'sections {sections}: {axes} even channel counts are wanted, at most {dim} together')
  bases = [float(b) for b in base] if isinstance(base, (tuple, list)) else [float(base)] * axes
  if len(bases) != axes or any(not (b > 0 and math.isfinite(b)) for b in bases):
    raise ValueError(f'base {base}: one positive number, or one per axis')
  return _Rotary.apply(x, positions.contiguous(), sections, bases, bool(interleaved))


# ------------------------------------------------------------------------------------------------- cross attention
def _attn_args(q, k, v, key_lengths, key_mask, scale):
  args = _ffi.TapirAttnArgs(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], scale)
  args.q, args.k, args.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
  args.q_stride[:], args.k_stride[:], args.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
  args.key_lengths, args.key_mask = _ptr(key_lengths), _ptr(key_mask)
  return args


def _attn_workspace(like, args, backward):
  nbytes = ctypes.c_uint64()
  _call(like, 'tapir_cross_attention_workspace', ctypes.byref(args), int(backward), ctypes.byref(nbytes), on_stream=False)
  work = _workspace(nbytes.value, like.device)
  args.workspace, args.workspace_bytes = _ptr(work), nbytes.value
  return work


class _CrossAttention(torch.autograd.Function):

  @staticmethod
  def forward(ctx, q, k, v, key_lengths, key_mask, scale, train):
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    args = _attn_args(q, k, v, key_lengths, key_mask, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    args.out = out.data_ptr()
    out32 = lse = None
    if train:
      out32 = torch.empty(q.shape, dtype=torch.float32, device=q.device)
      lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
      args.out_f32, args.lse = out32.data_ptr(), lse.data_ptr()
    work = _attn_workspace(q, args, False)  # (held until the call has been enqueued)
    _call(q, 'tapir_cross_attention', ctypes.byref(args))
    del work
    if train:
      ctx.save_for_backward(q, k, v, key_lengths, key_mask, out32, lse)
      ctx.scale = scale
    return out

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, dout):
    q, k, v, key_lengths, key_mask, out32, lse = ctx.saved_tensors
    dout = _aligned(dout)
    args = _attn_args(q, k, v, key_lengths, key_mask, ctx.scale)
    args.out_f32, args.lse = out32.data_ptr(), lse.data_ptr()
    args.dout, args.dout_stride[:] = dout.data_ptr(), dout.stride()[:3]
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    args.dq, args.dk, args.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    work = _attn_workspace(q, args, True)
    _call(q, 'tapir_cross_attention_backward', ctypes.byref(args))
    del work
    return dq, dk, dv, None, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
  """``softmax(scale q k^T) v``: query tokens (points) read an encoder's tokens (the cells of a clip or of one frame).

  q: float32 or bfloat16 ``[batch, queries, heads, dim]``; k, v: the same type, ``[batch, keys, kv_heads, dim]``; heads a
  multiple of kv_heads (query head j reads key head ``j // (heads // kv_heads)``), dim a multiple of 8 up to 128, any
  lengths from zero on, any strides (tensors whose rows are not dense or not at multiples of 16 bytes are copied).
  key_lengths: int32 ``[batch]``, the tokens of each clip (clamped to 0 .. keys; on the GPU, not read by the host).
  key_mask: bool ``[batch, keys]``, True where a token may be attended to.  Tokens outside either are not read: they may
  hold anything, and their gradients are zeros.  A query without any token gives zeros.  scale: positive, default
  ``dim ** -0.5``.

  Returns ``[batch, queries, heads, dim]`` in q's type.  Scores, statistics and sums are float32; in bfloat16 the
  probabilities (and in the gradient the scores' gradients) are rounded to bfloat16 on their way into the second product."""
  _check_tensor('q', q, 4)
  for name, t in (('k', k), ('v', v)):
    _check_tensor(name, t, 4, like=q)
    if t.dtype != q.dtype:
      raise ValueError(f'{name} is {t.dtype}, q is {q.dtype}')
  batch, _, heads, dim = q.shape
  keys, kv_heads = k.shape[1:3]
  if k.shape != v.shape or k.shape[0] != batch or k.shape[3] != dim:
    raise ValueError(f'k {list(k.shape)} and v {list(v.shape)} have to be [{batch}, keys, kv_heads, {dim}] both')
  if heads < 1 or kv_heads < 1 or heads % kv_heads:
    raise ValueError(f'{heads} query heads are not a multiple of {kv_heads} key heads')
  if not 8 <= dim <= 128 or dim % 8:
    raise ValueError(f'the head dimension has to be a multiple of 8 up to 128, not {dim}')
  if key_lengths is not None:
    _check_tensor('key_lengths', key_lengths, 1, like=q)
    if key_lengths.dtype != torch.int32 or key_lengths.shape[0] != batch:
      raise ValueError(f'key_lengths have to be int32 [{batch}], not {key_lengths.dtype} {list(key_lengths.shape)}')
    key_lengths = key_lengths.contiguous()
  if key_mask is not None:
    _check_tensor('key_mask', key_mask, 2, like=q)
    if key_mask.dtype != torch.bool or tuple(key_mask.shape) != (batch, keys):
      raise ValueError(f'key_mask has to be bool [{batch}, {keys}], not {key_mask.dtype} {list(key_mask.shape)}')
    key_mask = key_mask.contiguous()
  scale = dim ** -0.5 if scale is None else float(scale)
  if not (scale > 0 and math.isfinite(scale)):
    raise ValueError(f'scale has to be positive and finite, not {scale}')
  train = torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v))
  return _CrossAttention.apply(q, k, v, key_lengths, key_mask, scale, train)
