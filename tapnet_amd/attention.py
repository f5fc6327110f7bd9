"""Operators of a learned readout of a clip's feature grids: layer normalisation, rotary positions of several axes and
cross attention of point queries to feature tokens, with their gradients.

They stand beside the fixed readout of the TAPIR path (the cost volume and its soft arg max,
tapnet/models/tapir_model.py:399-471): ``TAPIR.get_feature_grids`` gives the tokens ``[batch, frames * h * w, channels]``
that points attend to, their (t, y, x) coordinates are the positions.  Everything runs in hand-written gfx950 kernels
through the C ABI (``include/tapir_hip.h``); there is no CPU fallback.  Element types are the engine's two, float32 and
bfloat16; sums, statistics and the parameters of a norm are float32 in both.

Calls are enqueued on the current stream of the tensors' device, whatever the current device is; nothing synchronises.
Scratch memory comes from torch's allocator, so calls on several streams and captured graphs do not share any.  A graph
may capture them once a call of the same element type has been made on the device (it prepares the library); a backward
pass is captured on a side stream, with no eager autograd graph of the same leaves alive (torch's autograd engine would
wait for the eager graph's stream inside the capture; refused where such a leaf is an operator's input).  No kernel uses
atomics: the same call gives the same bits, also where only some of the gradients are asked for.  Gradients are not
differentiable again, and forward-mode tangents are refused (RuntimeError).

The argument checks and autograd nodes are in ``csrc/torch_ops.cpp`` (built beside the library), which registers the operators with
torch's dispatcher as ``torch.ops.tapnet_amd``: ``torch.jit.trace`` and ``make_fx`` record them, fake tensors get their shapes.
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from tapnet_amd import _ffi

_OPS = None


def _ops():
  """The binding of the C ABI's operators to torch tensors.  Fails loudly when it has not been built."""
  global _OPS
  if _OPS is None:
    _ffi.load_library()
    try:
      from tapnet_amd import _torch_ops
    except ImportError as e:
      raise RuntimeError('tapnet_amd/_torch_ops.so does not load: build it with `python -c "import __graft_entry__ as g; '
                         f'g.build()"` ({e})') from e
    _OPS = _torch_ops
  return _OPS


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
  """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, as the norms of the PIPs mixer (scale only,
  tapnet/models/tapir_model.py:70-77) and of ExtraConvs (:176) have it, for any shape, and with gradients.

  x: float32 or bfloat16 ``[..., channels]`` of any strides, at most 2^30 channels.  weight, bias: float32 ``[channels]`` or None.  Statistics
  and sums are float32; the result has x's type.  Gradients of x (its type), weight and bias (float32)."""
  return _ops().layer_norm(x, weight, bias, eps)


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
  bases = list(base) if isinstance(base, (tuple, list)) else [base]
  return _ops().rotary_positions(x, positions, sections, bases, interleaved)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
  """``softmax(scale q k^T) v``: query tokens (points) read an encoder's tokens (the cells of a clip or of one frame).

  q: float32 or bfloat16 ``[batch, queries, heads, dim]``; k, v: the same type, ``[batch, keys, kv_heads, dim]``; heads a
  multiple of kv_heads (query head j reads key head ``j // (heads // kv_heads)``), dim a multiple of 8 up to 128, any
  lengths from zero on, any strides (tensors whose rows are not dense or not at multiples of 16 bytes are copied).
  key_lengths: int32 ``[batch]``, the tokens of each clip (clamped to 0 .. keys; on the GPU, not read by the host).
  key_mask: bool ``[batch, keys]``, True where a token may be attended to.  Tokens outside either are not read: they may
  hold anything, and their gradients are zeros.  A query without any token gives zeros; one whose tokens' scores are all -inf, or hold a
  NaN or +inf, gives NaN, as softmax does.  scale: 2^-60 to 2^60, default ``dim ** -0.5``.

  Returns ``[batch, queries, heads, dim]`` in q's type.  Scores, statistics and sums are float32; in bfloat16 the
  probabilities and the scores' gradients enter the second products with 16 bits, twice bfloat16's eight.
  In float32 the result itself is kept for the backward pass, as softmax keeps its own: overwriting it in place is an error there.
  The gradients of q and k use the rounded result (``sum(grad * out)`` of a row): in float32, where one token dominates a row, they
  are up to 2.2 times as far from the exact ones as a form that sums over the tokens again, some 1e-6 of their size."""
  return _ops().cross_attention(q, k, v, key_lengths, key_mask, scale)
