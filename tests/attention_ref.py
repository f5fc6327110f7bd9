"""TEST INFRASTRUCTURE ONLY: layer normalisation, rotary positions and cross attention in 64 bits, from their formulas,
with bounds on how far the kernels' results may be off.

Every bound counts roundings: u = 2^-24 is half a step of float32 (every float32 operation is off by at most u of its result,
a sum of n terms by at most n u of the sum of their magnitudes, in whatever order), `unit(dtype)` half a step of the element
type (operands and results that are rounded to it).  All functions take and return torch tensors (any device)."""
import math

import torch

U = 2.0 ** -24


def unit(dtype):
  return torch.finfo(dtype).eps / 2


def rounded(value, error, dtype):
  """Bound of a result whose float32 value is `value` within `error`, after rounding to `dtype` (f32: the last operation's)."""
  tiny = torch.finfo(dtype).tiny * unit(dtype) if dtype == torch.bfloat16 else 1e-38
  return error + unit(dtype) * (value.abs() + error) + tiny


# ------------------------------------------------------------------------------------------------------- layer norm
def layer_norm(x, weight, bias, eps, dy=None):
  """-> [(value, bound)] of y, and with dy of dx, dweight, dbias (None where there is no parameter)."""
  dtype, n = x.dtype, x.shape[-1]
  x = x.double()
  w = torch.ones(n, dtype=x.dtype, device=x.device) if weight is None else weight.double()
  b = torch.zeros(n, dtype=x.dtype, device=x.device) if bias is None else bias.double()
  mean = x.mean(-1, keepdim=True)
  c = x - mean
  var = (c * c).mean(-1, keepdim=True)
  r = 1 / torch.sqrt(var + eps)
  e_mean = (n + 2) * U * x.abs().mean(-1, keepdim=True)
  e_c = e_mean + U * c.abs()
  e_var = (n + 3) * U * (var + e_mean ** 2) + 2 * (c.abs() * e_c).mean(-1, keepdim=True) + (e_c ** 2).mean(-1, keepdim=True)
  e_r = 0.5 * e_var / torch.clamp(var + eps - e_var, min=1e-300) + 4 * U          # relative, of rstd
  un = c * r
  e_un = e_c * r * (1 + e_r) + un.abs() * (e_r + 2 * U)
  y = un * w + b
  out = [(y, rounded(y, e_un * w.abs() + 2 * U * (un * w).abs(), dtype))]
  if dy is None:
    return out
  dy = dy.double()
  g = dy * w
  m1, m2 = g.mean(-1, keepdim=True), (g * un).mean(-1, keepdim=True)
  e1 = (n + 2) * U * g.abs().mean(-1, keepdim=True)
  e2 = (n + 3) * U * (g * un).abs().mean(-1, keepdim=True) + (g.abs() * e_un).mean(-1, keepdim=True)
  inner = g - m1 - un * m2
  e_in = 4 * U * (g.abs() + m1.abs() + (un * m2).abs()) + e1 + un.abs() * e2 + m2.abs() * e_un + e_un * e2
  dx = r * inner
  out.append((dx, rounded(dx, r * (1 + e_r) * e_in + dx.abs() * (e_r + U), dtype)))
  rows = x.numel() // n
  flat = lambda t: t.reshape(-1, n)
  terms = flat(dy * un)
  out.append(None if weight is None else
             (terms.sum(0), (rows + 4) * U * terms.abs().sum(0) + flat(dy.abs() * e_un).sum(0) + 1e-38))
  out.append(None if bias is None else (flat(dy).sum(0), (rows + 2) * U * flat(dy).abs().sum(0) + 1e-38))
  return out


# ------------------------------------------------------------------------------------------------- rotary positions
def rotary(x, positions, sections, bases, interleaved, inverse=False):
  """-> (value, bound).  Angle: 2 pi times a fraction of a turn that is rounded to float32 once (2 pi 2^-26 < 1.6 u); reduced to
  a quarter turn without error, times 2 pi (u pi / 4 each for the product and the constant); the polynomials add a few u: sine
  and cosine are off by less than 8 u."""
  dtype = x.dtype
  x = x.double()
  out, err = x.clone(), torch.zeros_like(x)
  begin = 0
  for a, (width, base) in enumerate(zip(sections, bases)):
    i = torch.arange(width // 2, device=x.device)
    lo = begin + (2 * i if interleaved else i)
    hi = lo + 1 if interleaved else lo + width // 2
    angle = positions[..., a, None].double() * base ** (-2.0 * i.double() / max(width, 1))
    angle = (-angle if inverse else angle).unsqueeze(-2)
    cos, sin = angle.cos(), angle.sin()
    p, q = x[..., lo], x[..., hi]
    out[..., lo], out[..., hi] = p * cos - q * sin, p * sin + q * cos
    both = (p.abs() + q.abs()) * 10 * U
    err[..., lo], err[..., hi] = both, both
    begin += width
  return out, rounded(out, err, dtype)


# -------------------------------------------------------------------------------------------------- cross attention
def attention(q, k, v, keep, scale, dout=None):
  """-> [(value, bound)] of out, and with dout of dq, dk, dv.  keep: bool [batch, keys]."""
  dtype = q.dtype
  h = 0.0 if dtype == torch.float32 else unit(dtype)          # rounding of the second products' operands
  batch, queries, heads, dim = q.shape
  keys, kv_heads = k.shape[1:3]
  group = heads // kv_heads
  rows = lambda t: t.double().reshape(batch, queries, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(
      batch, kv_heads, group * queries, dim)
  back = lambda t: t.reshape(batch, kv_heads, group, queries, dim).permute(0, 3, 1, 2, 4).reshape(batch, queries, heads, dim)
  gone = ~keep[:, None, :, None]
  kk = k.double().permute(0, 2, 1, 3).masked_fill(gone, 0.0)
  vv = v.double().permute(0, 2, 1, 3).masked_fill(gone, 0.0)
  qq = rows(q)
  kt, vt = kk.transpose(2, 3).contiguous(), vv.transpose(2, 3).contiguous()
  raw = qq @ kt
  s = (raw * scale).masked_fill(gone.transpose(2, 3), -math.inf)
  top = s.amax(-1, keepdim=True) if keys else torch.full(s.shape[:-1] + (1,), -math.inf, dtype=s.dtype, device=s.device)
  top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
  p = torch.exp(s - top)
  total = p.sum(-1, keepdim=True)
  p = p / torch.where(total == 0, torch.ones_like(total), total)
  o = p @ vv
  # a probability: the score (dim + 2 roundings of its products, two of the scale), the exponent's own rounding, the maximum or
  # L_r (as far off as the scores, plus the sum's n roundings), the exponential (2 steps)
  absraw = qq.abs() @ kt.abs()
  e_s = ((dim + 4) * U * absraw * scale).amax(-1, keepdim=True) if keys else torch.zeros_like(top)
  big = torch.maximum(s.masked_fill(gone.transpose(2, 3), 0.0).abs().amax(-1, keepdim=True), top.abs()) if keys else top.abs()
  e_p = 2 * e_s + 6 * U * (big + math.log(max(keys, 1)) + 1) + (keys + 12) * U
  # (exp2 gives zero below 2^-126, and products may take operands below it as zero: an absolute error of that size each)
  low = 2.0 ** -125
  absum = p @ vv.abs()
  ones = torch.ones_like(p)
  e_o32 = absum * (2 * e_p + (keys + 6) * U + 2 * h) + low * (ones @ vv.abs())   # (h: the operand and the sum of its roundings)
  out = [(back(o), rounded(back(o), back(e_o32), dtype))]
  if dout is None:
    return out
  do = rows(dout)
  dp = do @ vt
  e_dp = (dim + 2) * U * (do.abs() @ vt.abs())
  dot = (do * o).sum(-1, keepdim=True)
  e_dot = (dim + 2) * U * (do.abs() * o.abs()).sum(-1, keepdim=True) + (do.abs() * e_o32).sum(-1, keepdim=True)
  ds = p * (dp - dot)
  e_ds = p * (e_p * (1 + e_p) * ((dp - dot).abs() + e_dp + e_dot) + e_dp + e_dot + 3 * U * (dp.abs() + dot.abs()))
  e_ds = e_ds + h * (ds.abs() + e_ds) + low * (1 + dp.abs() + dot.abs())
  n_rows = group * queries
  dq = scale * (ds @ kk)
  e_dq = scale * (e_ds @ kk.abs() + (keys + 4) * U * ((ds.abs() + e_ds) @ kk.abs()))
  dst, pt = ds.transpose(2, 3).contiguous(), p.transpose(2, 3).contiguous()
  dk = scale * (dst @ qq)
  e_dk = scale * (e_ds.transpose(2, 3).contiguous() @ qq.abs() + (n_rows + 4) * U * (dst.abs() @ qq.abs()) * 1.01)
  dv = pt @ do
  e_dv = (pt * (e_p.transpose(2, 3) + h + (n_rows + 4) * U) * 1.01 + low) @ do.abs()
  out.append((back(dq), rounded(back(dq), back(e_dq), dtype)))
  for t, e in ((dk, e_dk), (dv, e_dv)):
    t, e = t.permute(0, 2, 1, 3), e.permute(0, 2, 1, 3)
    out.append((t, rounded(t, e, dtype)))
  return out


def check(name, got, want):
  """`got` within the bound of want = (value, bound) everywhere; a failure says where and by how much."""
  value, bound = want
  assert tuple(got.shape) == tuple(value.shape), f'{name}: shape {tuple(got.shape)}, not {tuple(value.shape)}'
  if value.numel() == 0:
    return
  diff = (got.double() - value).abs()
  ratio = torch.where(diff == 0, torch.zeros_like(diff), diff / bound)
  ratio = torch.where(torch.isnan(ratio), torch.full_like(ratio, math.inf), ratio)
  worst = int(ratio.argmax())
  at = [int(i) for i in torch.unravel_index(torch.tensor(worst), value.shape)]
  r = float(ratio.flatten()[worst])
  assert r <= 1, (f'{name}{at}: {float(got.flatten()[worst])} for {float(value.flatten()[worst])}, '
                  f'{r:.3g} times the bound {float(bound.flatten()[worst]):.3g}; '
                  f'{int((ratio > 1).sum())} of {ratio.numel()} outside')
