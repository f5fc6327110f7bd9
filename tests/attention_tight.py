"""TEST INFRASTRUCTURE ONLY: cross attention in 64 bits with bounds that stay narrow over many keys, and inputs whose tokens each
show in a result.

tests/attention_ref.py counts every rounding at its worst, all of one sign: n terms are off by n u of their magnitudes.  Roundings
are of either sign.  Each is at most u and has no preferred sign, so (Azuma's inequality) a sum of n of them, of sizes c_i, stays
below lambda sqrt(sum c_i^2) except with probability 2 exp(-lambda^2 / 2); lambda = 8 here, below 3e-14 an element.  Hence

* a sum of n terms with partial sums S_i is off by at most lambda sqrt(n) u max|S_i| (`count(n)` max|S_i|; n + 4 where that is
  less).  Terms of either sign, as the inputs here have them, walk at random: max|S_i| <= |S_n| + 4 sqrt(sum of squares);
* errors of the terms (scores, rounded operands) add up by their squares; what a whole row shares (the error of its maximum and
  sum, of D) is a factor of the row's result, or of sum p k.

The bf16 operands of the second products are taken at two parts: the upper one, truncated to 8 significant bits, leaves less
than 2^-7, of which the lower one, rounded, loses 2^-8 at most."""
import math

import torch

from tests.attention_ref import U, check

LAMBDA = 8.0
TWO_PARTS = 2.0 ** -15
LOW = 2.0 ** -125        # exp2 gives zero below 2^-126, and products may take operands below it as zero


def count(n):
  return min(n + 4, LAMBDA * math.sqrt(n + 4)) * U


def rounded(value, error, dtype):
  """Bound of a result that is `value` within `error` before it is rounded: half a step of `dtype` where it lies (at most
  finfo.eps / 2 of the value, half of that below the next power of two)."""
  info = torch.finfo(dtype)
  size = torch.clamp(value.abs() + error, min=info.tiny)
  return error + torch.exp2(torch.floor(torch.log2(size))) * (info.eps / 2) + info.tiny * info.eps


def attention(q, k, v, keep, scale, dout=None):
  """-> [(value, bound)] of the unrounded out (f32), of out, and with dout of dq, dk, dv.  keep: bool [batch, keys]."""
  dtype = q.dtype
  h = 0.0 if dtype == torch.float32 else TWO_PARTS
  batch, queries, heads, dim = q.shape
  keys, kv_heads = k.shape[1:3]
  group = heads // kv_heads
  rows = lambda t: t.double().reshape(batch, queries, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(
      batch, kv_heads, group * queries, dim)
  back = lambda t: t.reshape(batch, kv_heads, group, queries, dim).permute(0, 3, 1, 2, 4).reshape(batch, queries, heads, dim)
  turned = lambda t: t.transpose(2, 3).contiguous()
  gone = ~keep[:, None, :, None]
  kk = k.double().permute(0, 2, 1, 3).masked_fill(gone, 0.0)
  vv = v.double().permute(0, 2, 1, 3).masked_fill(gone, 0.0)
  qq = rows(q)
  s = (qq @ turned(kk) * scale).masked_fill(turned(gone), -math.inf)
  top = s.amax(-1, keepdim=True)
  top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
  p = torch.exp(s - top)
  total = p.sum(-1, keepdim=True)
  safe = torch.where(total == 0, torch.ones_like(total), total)
  p = p / safe
  o = p @ vv
  # what the exponential gets: the score (its products may start at L, m + log l over the scale), the scale's and the
  # exponent's roundings; then the exponential (2 u) and its factors.  A row shares the error of its sum.
  size = s.masked_fill(turned(gone), 0.0).abs()
  big = top.abs() + safe.log().abs()
  e_x = count(dim) * (qq.abs() @ turned(kk.abs()) * scale + big) + 4 * U * (size + big) + 8 * U
  e_row = (p * e_x).square().sum(-1, keepdim=True).sqrt() + count(keys) + 4 * U
  own = e_x.square() + (LAMBDA * h) ** 2                       # of p, relative, squared
  walk = lambda total, squares, n: count(n) * (total.abs() + 4 * squares.sqrt())
  p2, v2, k2, q2 = p.square(), vv.square(), kk.square(), qq.square()
  e_o = o.abs() * e_row + ((p2 * own) @ v2).sqrt() + walk(o, p2 @ v2, keys) + LOW * vv.abs().sum(2, keepdim=True)
  out = [(back(o), rounded(back(o), back(e_o), torch.float32)), (back(o), rounded(back(o), back(e_o), dtype))]
  if dout is None:
    return out
  do = rows(dout)
  dp = do @ turned(vv)
  dot = (do * o).sum(-1, keepdim=True)
  e_dp = count(dim) * (do.abs() @ turned(vv.abs()) + dot.abs())
  e_dot = count(dim) * (do.abs() * o.abs()).sum(-1, keepdim=True) + (do.abs() * (e_o + U * o.abs())).sum(-1, keepdim=True)
  ds = p * (dp - dot)
  ds2 = ds.square()
  own_ds = p2 * (e_x.square() * (dp - dot).square() + e_dp.square() + (3 * U * (dp.abs() + dot.abs())).square()) + ds2 * (LAMBDA * h) ** 2
  low = LOW * (1 + dp.abs() + dot.abs())
  dq = scale * (ds @ kk)
  e_dq = (dq.abs() * e_row + scale * ((own_ds @ k2).sqrt() + e_dot * (p @ kk).abs() + low @ kk.abs())
          + walk(dq, scale ** 2 * (ds2 @ k2), keys)) * 1.01
  n = group * queries
  shared = own_ds + ds2 * e_row.square() + p2 * e_dot.square()
  dk = scale * (turned(ds) @ qq)
  e_dk = (scale * ((turned(shared) @ q2).sqrt() + turned(low) @ qq.abs()) + walk(dk, scale ** 2 * (turned(ds2) @ q2), n)) * 1.01
  dv = turned(p) @ do
  do2 = do.square()
  e_dv = ((turned(p2 * (own + e_row.square())) @ do2).sqrt() + LOW * do.abs().sum(2, keepdim=True) + walk(dv, turned(p2) @ do2, n)) * 1.01
  out.append((back(dq), rounded(back(dq), back(e_dq), dtype)))
  for t, e in ((dk, e_dk), (dv, e_dv)):
    t, e = t.permute(0, 2, 1, 3), e.permute(0, 2, 1, 3)
    out.append((t, rounded(t, e, dtype)))
  return out


def picked(keys, most):
  """Tokens that each have a query of their own: the last one, both ends of tiles of 32, 64 and 128, the others in equal steps."""
  ends = {keys - 1, 0}
  for tile in (32, 64, 128):
    last = (keys - 1) // tile * tile                # the first of the last, unfinished tile
    ends |= {t for t in (last, last - 1, tile - 1, tile) if 0 <= t < keys}
  rest = max(0, most - len(ends))
  ends |= {i * keys // rest for i in range(rest)} if rest else set()
  return sorted(ends)


def dominated(gen, dtype, device, keys, heads, kv_heads, dim, most=96, scale=None):
  """One query for each of some tokens, whose probability is near 9 / 10 for it: a token, tile or split that is lost or counted
  twice moves a result by its own size.  Scores of the other keys have a deviation of about 1 + ln(keys) / 4."""
  randn = lambda *shape: torch.randn(*shape, generator=gen, device=device)
  at = torch.tensor(picked(keys, most), device=device)
  k, v = randn(1, keys, kv_heads, dim), randn(1, keys, kv_heads, dim)
  k = k / k.norm(dim=-1, keepdim=True)
  scale = dim ** -0.5 if scale is None else scale
  q = (k[:, at] * (math.log(keys) + 2.2) / scale).repeat_interleave(heads // kv_heads, 2)
  return q.to(dtype), k.to(dtype), v.to(dtype), randn(1, len(at), heads, dim).to(dtype), at


__all__ = ['attention', 'check', 'count', 'dominated', 'picked']
