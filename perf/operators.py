"""Cases for the operators of `tapnet_amd.attention`: layer normalisation, rotary positions of several axes and
cross attention of point queries to a clip's feature tokens, each forward alone or with its gradients.

`run` computes a case in plain torch operations, or, where `own` is set, through the framework's entry points.
A clip of 48 frames has 32 x 32 cells of 256 channels a frame (49152 tokens), the online model sees one frame
(1024 tokens) at a time, and 256 to 4096 points are tracked.
"""
import math

import torch

own = False

EPS = 1e-5
BASE = 10000.0


def listed():
  return [
      # the tokens of one frame of the online model, normalised on their way into a projection: a latency
      {'name': 'norm_frame_bf16', 'op': 'norm', 'dtype': 'bf16', 'rows': 1024, 'channels': 256, 'affine': 'full',
       'train': False},
      # all feature tokens of a clip in a training step, with both parameters' gradients
      {'name': 'norm_train_clip_bf16', 'op': 'norm', 'dtype': 'bf16', 'rows': 49152, 'channels': 256,
       'affine': 'full', 'train': True},
      # 256 points x 48 frames of the mixer's 512 channels, scale only as in the mixer's norms
      {'name': 'norm_train_mixer_f32', 'op': 'norm', 'dtype': 'f32', 'rows': 12288, 'channels': 512,
       'affine': 'scale', 'train': True},
      # the positions (t, y, x) of 256 query points put into their 8 heads: a latency
      {'name': 'rope_points_bf16', 'op': 'rope', 'dtype': 'bf16', 'batch': 1, 'tokens': 256, 'heads': 8, 'dim': 32,
       'axes': 3, 'interleaved': False, 'shared': False, 'train': False},
      # the cells of a whole clip, the same positions for both clips of the batch
      {'name': 'rope_train_clip_bf16', 'op': 'rope', 'dtype': 'bf16', 'batch': 2, 'tokens': 49152, 'heads': 4,
       'dim': 64, 'axes': 3, 'interleaved': False, 'shared': True, 'train': True},
      # image positions (y, x), neighbouring channels as pairs, sizes that fit no tile
      {'name': 'rope_train_image_f32', 'op': 'rope', 'dtype': 'f32', 'batch': 3, 'tokens': 4095, 'heads': 6,
       'dim': 40, 'axes': 2, 'interleaved': True, 'shared': False, 'train': True},
      # the online model: 256 points read the frame that has just come
      {'name': 'attend_frame_bf16', 'op': 'attend', 'dtype': 'bf16', 'batch': 1, 'queries': 256, 'keys': 1024,
       'heads': 8, 'kv_heads': 8, 'dim': 32, 'padding': 'none', 'packed': True, 'train': False},
      # one new point reads a whole clip, four query heads to a key head
      {'name': 'attend_one_query_bf16', 'op': 'attend', 'dtype': 'bf16', 'batch': 1, 'queries': 1, 'keys': 49152,
       'heads': 8, 'kv_heads': 2, 'dim': 64, 'padding': 'none', 'packed': False, 'train': False},
      # 4096 points read a whole clip
      {'name': 'attend_points_bf16', 'op': 'attend', 'dtype': 'bf16', 'batch': 1, 'queries': 4096, 'keys': 49152,
       'heads': 4, 'kv_heads': 4, 'dim': 64, 'padding': 'none', 'packed': True, 'train': False},
      # a training step of 256 points on a whole clip
      {'name': 'attend_train_clip_bf16', 'op': 'attend', 'dtype': 'bf16', 'batch': 1, 'queries': 256, 'keys': 49152,
       'heads': 4, 'kv_heads': 4, 'dim': 64, 'padding': 'none', 'packed': True, 'train': True},
      # a training step on clips of different lengths, padded to the longest, with shared key heads
      {'name': 'attend_train_ragged_bf16', 'op': 'attend', 'dtype': 'bf16', 'batch': 3, 'queries': 1000,
       'keys': 8200, 'heads': 4, 'kv_heads': 2, 'dim': 128, 'padding': 'lengths', 'packed': False, 'train': True},
      # the same in full precision on a few frames of which some cells are masked out
      {'name': 'attend_train_masked_f32', 'op': 'attend', 'dtype': 'f32', 'batch': 2, 'queries': 256, 'keys': 4096,
       'heads': 8, 'kv_heads': 8, 'dim': 32, 'padding': 'mask', 'packed': False, 'train': True},
  ]


def _spread(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  op = rng.choice(['norm', 'rope', 'attend', 'attend'])
  dtype = rng.choice(['bf16', 'f32'])
  train = rng.random() < 0.5
  if op == 'norm':
    return {'op': op, 'dtype': dtype, 'rows': _spread(rng, 1, 49152), 'channels': _spread(rng, 8, 1024),
            'affine': rng.choice(['full', 'scale', 'none']), 'train': train}
  if op == 'rope':
    return {'op': op, 'dtype': dtype, 'batch': rng.randint(1, 3), 'tokens': _spread(rng, 1, 16384),
            'heads': rng.randint(1, 8), 'dim': 2 * rng.randint(3, 64), 'axes': rng.randint(1, 3),
            'interleaved': rng.random() < 0.5, 'shared': rng.random() < 0.5, 'train': train}
  kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
  case = {'op': op, 'dtype': dtype, 'batch': rng.randint(1, 3), 'queries': _spread(rng, 1, 4096),
          'keys': _spread(rng, 8 if train else 1, 49152), 'heads': kv_heads * group, 'kv_heads': kv_heads,
          'dim': 8 * rng.randint(1, 16), 'padding': rng.choice(['none', 'lengths', 'lengths', 'mask']),
          'packed': rng.random() < 0.5, 'train': train}
  # (a row that attends to a single key has gradients of exactly zero, in which nothing can be compared: training
  # starts at 8 keys)  No more work than a training step of 1024 points on 12288 tokens
  most = 1024 * 12288 * 4 * 64 * 14
  while True:
    cost = case['batch'] * case['heads'] * case['queries'] * case['keys'] * case['dim'] * 14
    if cost <= most:
      return case
    case['queries' if case['queries'] > case['keys'] else 'keys'] = max(case['queries'], case['keys']) // 2 + 1


def _type(case):
  return torch.bfloat16 if case['dtype'] == 'bf16' else torch.float32


def _lengths(case):
  """Tokens of each clip of a padded batch: the first is whole, the last of three has none."""
  return [case['keys'], (case['keys'] + 1) // 2, 0][:case['batch']]


def _sections(case):
  """Channels of each axis of a head: equal shares, what is left over goes to the first ones a pair at a time."""
  pairs, axes = case['dim'] // 2, case['axes']
  return tuple(2 * (pairs // axes + (a < pairs % axes)) for a in range(axes))


def prepare(case, seed):
  gen = torch.Generator(device='cuda').manual_seed(seed)
  dtype = _type(case)

  def randn(*shape):
    return torch.randn(*shape, generator=gen, device='cuda')

  def leaf(t):
    return t.detach().requires_grad_(case['train'])

  state = {'case': case}
  if case['op'] == 'norm':
    rows, channels = case['rows'], case['channels']
    # activations of unlike rows: a mean of their own each, spread between a tenth and some units
    x = randn(rows, channels) * torch.exp(randn(rows, 1)) + randn(rows, 1)
    state['x'] = leaf(x.to(dtype))
    state['weight'] = leaf(1 + 0.2 * randn(channels)) if case['affine'] != 'none' else None
    state['bias'] = leaf(0.2 * randn(channels)) if case['affine'] == 'full' else None
    if case['train']:
      state['dy'] = randn(rows, channels).to(dtype)
  elif case['op'] == 'rope':
    batch, tokens, heads, dim, axes = (case[n] for n in ('batch', 'tokens', 'heads', 'dim', 'axes'))
    state['x'] = leaf(randn(batch, tokens, heads, dim).to(dtype))
    # points anywhere in 48 frames of 256 x 256 pixels: (t, y, x), (y, x), or the frame of a long video alone
    sizes = {1: [100000.], 2: [256., 256.], 3: [48., 256., 256.]}[axes]
    shape = (tokens, axes) if case['shared'] else (batch, tokens, axes)
    state['positions'] = torch.rand(*shape, generator=gen, device='cuda') * torch.tensor(sizes, device='cuda')
    if axes != 2:
      state['positions'][..., 0].floor_()
    state['sections'] = _sections(case)
    if case['train']:
      state['dy'] = randn(batch, tokens, heads, dim).to(dtype)
  else:
    batch, queries, keys, heads, kv_heads, dim = (
        case[n] for n in ('batch', 'queries', 'keys', 'heads', 'kv_heads', 'dim'))
    # keys and values as one projection leaves them, or each in a tensor of its own
    if case['packed']:
      k, v = randn(batch, keys, 2, kv_heads, dim).to(dtype).unbind(2)
    else:
      k, v = randn(batch, keys, kv_heads, dim).to(dtype), randn(batch, keys, kv_heads, dim).to(dtype)
    # every second query resembles one of the keys, as a tracked point does its place in a frame
    q = randn(batch, queries, heads, dim)
    pick = torch.randint(0, keys, (queries,), generator=gen, device='cuda')
    like = k[:, pick].float().repeat_interleave(heads // kv_heads, dim=2)
    q[:, 1::2] = 0.5 * q[:, 1::2] + like[:, 1::2]
    state.update(q=leaf(q.to(dtype)), k=leaf(k), v=leaf(v), key_lengths=None, key_mask=None)
    if case['padding'] == 'lengths':
      state['key_lengths'] = torch.tensor(_lengths(case), dtype=torch.int32, device='cuda')
    elif case['padding'] == 'mask':
      state['key_mask'] = torch.rand(batch, keys, generator=gen, device='cuda') < 0.75
    if case['train']:
      state['dy'] = randn(batch, queries, heads, dim).to(dtype)
  return state


def work(case):
  size = 2 if case['dtype'] == 'bf16' else 4
  if case['op'] == 'norm':
    n = case['rows'] * case['channels']
    params = 4 * case['channels'] * {'full': 2, 'scale': 1, 'none': 0}[case['affine']]
    if case['train']:  # x and dy read, y and dx written; the parameters and their gradients
      return {'bytes': 4 * n * size + 2 * params, 'flops': 20 * n}
    return {'bytes': 2 * n * size + params, 'flops': 8 * n}
  if case['op'] == 'rope':
    n = case['batch'] * case['tokens'] * case['heads'] * case['dim']
    positions = 4 * case['tokens'] * case['axes'] * (1 if case['shared'] else case['batch'])
    passes = 2 if case['train'] else 1
    return {'bytes': 2 * passes * n * size + positions, 'flops': 3 * passes * n}
  kept = {'none': case['batch'] * case['keys'], 'lengths': sum(_lengths(case)),
          'mask': round(0.75 * case['batch'] * case['keys'])}[case['padding']]
  pairs = case['heads'] * case['queries'] * kept
  q = case['batch'] * case['queries'] * case['heads'] * case['dim'] * size
  kv = kept * case['kv_heads'] * case['dim'] * size
  masks = {'none': 0, 'lengths': 4 * case['batch'], 'mask': case['batch'] * case['keys']}[case['padding']]
  if case['train']:  # q, k, v and dy read; the output and three gradients written, the padding's zeros too
    dkv = case['batch'] * case['keys'] * case['kv_heads'] * case['dim'] * size
    return {'bytes': 4 * q + 2 * kv + 2 * dkv + masks, 'flops': 14 * pairs * case['dim']}
  return {'bytes': 2 * q + 2 * kv + masks, 'flops': 4 * pairs * case['dim']}


def run(state):
  case = state['case']
  if own:
    return _framework(state)
  with torch.no_grad():
    return {'norm': _plain_norm, 'rope': _plain_rope, 'attend': _plain_attend}[case['op']](state)


def _framework(state):
  """The calls of a user's program; gradients through autograd, as a training step takes them."""
  from tapnet_amd import attention
  case = state['case']
  with torch.set_grad_enabled(case['train']):
    if case['op'] == 'norm':
      inputs = [t for t in (state['x'], state['weight'], state['bias']) if t is not None]
      y = attention.layer_norm(state['x'], state['weight'], state['bias'], eps=EPS)
    elif case['op'] == 'rope':
      inputs = [state['x']]
      y = attention.rotary_positions(state['x'], state['positions'], sections=state['sections'], base=BASE,
                                     interleaved=case['interleaved'])
    else:
      inputs = [state['q'], state['k'], state['v']]
      y = attention.cross_attention(state['q'], state['k'], state['v'], key_lengths=state['key_lengths'],
                                    key_mask=state['key_mask'])
    if not case['train']:
      return [y]
    return [y.detach(), *torch.autograd.grad(y, inputs, state['dy'])]


def _plain_norm(state):
  x, weight, bias = state['x'].float(), state['weight'], state['bias']
  dtype = state['x'].dtype
  centred = x - x.mean(-1, keepdim=True)
  rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
  unit = centred * rstd
  y = unit if weight is None else unit * weight
  if bias is not None:
    y = y + bias
  if not state['case']['train']:
    return [y.to(dtype)]
  dy = state['dy'].float()
  g = dy if weight is None else dy * weight
  dx = rstd * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))
  grads = [dx.to(dtype)]
  if weight is not None:
    grads.append((dy * unit).sum(0))
  if bias is not None:
    grads.append(dy.sum(0))
  return [y.to(dtype), *grads]


def _plain_rope(state):
  case = state['case']
  # the axis and the frequency of every pair of channels; angles in 64 bits
  sections = torch.tensor(state['sections'], device='cuda')
  axis = torch.repeat_interleave(torch.arange(case['axes'], device='cuda'), sections // 2,
                                 output_size=case['dim'] // 2)
  first = (torch.cumsum(sections // 2, 0) - sections // 2)[axis]
  pair = torch.arange(case['dim'] // 2, device='cuda') - first
  frequency = torch.exp(-math.log(BASE) * 2.0 * pair.double() / sections[axis])
  angle = state['positions'].double()[..., axis] * frequency
  cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
  # the two channels of every pair: neighbours, or the halves of the axis' section
  low = 2 * first + (2 * pair if case['interleaved'] else pair)
  high = low + (1 if case['interleaved'] else sections[axis] // 2)

  def turn(x, sin):
    a, b = x.float()[..., low], x.float()[..., high]
    out = torch.empty_like(x)
    out[..., low] = (a * cos - b * sin).to(x.dtype)
    out[..., high] = (a * sin + b * cos).to(x.dtype)
    return out

  y = turn(state['x'], sin)
  return [y, turn(state['dy'], -sin)] if case['train'] else [y]


def _plain_attend(state):
  case = state['case']
  batch, queries, keys, heads, kv_heads, dim = (
      case[n] for n in ('batch', 'queries', 'keys', 'heads', 'kv_heads', 'dim'))
  group, dtype, scale = heads // kv_heads, state['q'].dtype, 1 / math.sqrt(dim)

  def rows(t):  # [batch, queries, heads, dim] -> [batch, kv_heads, group * queries, dim]
    return t.float().view(batch, queries, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(
        batch, kv_heads, group * queries, dim)

  def back(t):
    return t.view(batch, kv_heads, group, queries, dim).permute(0, 3, 1, 2, 4).reshape(
        batch, queries, heads, dim).to(dtype)

  q = rows(state['q'])
  k, v = (state[n].float().transpose(1, 2).contiguous() for n in 'kv')
  scores = torch.matmul(q, k.transpose(2, 3)).mul_(scale)
  keep = state['key_mask']
  if state['key_lengths'] is not None:
    keep = torch.arange(keys, device='cuda') < state['key_lengths'][:, None]
  if keep is not None:
    scores.masked_fill_(~keep[:, None, None, :], -math.inf)
  top = scores.amax(-1, keepdim=True)
  p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
  total = p.sum(-1, keepdim=True)
  p.div_(torch.where(total == 0, 1.0, total))
  out = back(torch.matmul(p, v))
  if not case['train']:
    return [out]
  dy = rows(state['dy'])
  dv = torch.matmul(p.transpose(2, 3), dy)
  dp = torch.matmul(dy, v.transpose(2, 3))
  ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(scale)
  dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
  return [out, back(dq), *(t.transpose(1, 2).to(dtype) for t in (dk, dv))]


def exact(case, seed):
  state = prepare(case, seed)
  with torch.no_grad():
    if case['op'] == 'norm':
      return _exact_norm(state)
    if case['op'] == 'rope':
      return _exact_rope(state)
    return _exact_attend(state)


def _exact_norm(state):
  x = state['x'].double()
  weight = state['weight'].double() if state['weight'] is not None else torch.ones_like(x[0])
  bias = state['bias'].double() if state['bias'] is not None else torch.zeros_like(x[0])
  sigma = torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + EPS)
  unit = (x - x.mean(-1, keepdim=True)) / sigma
  out = [weight * unit + bias]
  if state['case']['train']:
    # the Jacobian of a row: (1 - 1/C - unit unit^T / C) / sigma
    dy, channels = state['dy'].double(), x.shape[1]
    g = dy * weight
    along = torch.einsum('rc,rc->r', g, unit)[:, None] / channels
    out.append((g - g.sum(-1, keepdim=True) / channels - along * unit) / sigma)
    if state['weight'] is not None:
      out.append(torch.einsum('rc,rc->c', dy, unit))
    if state['bias'] is not None:
      out.append(torch.einsum('rc->c', dy))
  return out


def _exact_rope(state):
  """Every pair as a complex number, turned by exp(i angle), axis after axis."""
  case = state['case']

  def turn(x, sign):
    parts, begin = [], 0
    for a, width in enumerate(state['sections']):
      part = x[..., begin:begin + width].double()
      begin += width
      if width == 0:
        continue
      power = torch.arange(0, width, 2, device='cuda').double() / width
      angle = sign * state['positions'][..., a, None].double() / BASE ** power
      e = torch.polar(torch.ones_like(angle), angle).unsqueeze(-2)
      if case['interleaved']:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], width // 2, 2).contiguous()) * e
        parts.append(torch.view_as_real(z).flatten(-2))
      else:
        z = torch.complex(part[..., :width // 2], part[..., width // 2:]) * e
        parts.append(torch.cat([z.real, z.imag], -1))
    return torch.cat(parts, -1)

  out = [turn(state['x'], 1.0)]
  return out + [turn(state['dy'], -1.0)] if case['train'] else out


def _exact_attend(state):
  """Head by head, some query rows at a time; masked keys are left out of the sums."""
  case = state['case']
  q, k, v = (state[n].detach() for n in 'qkv')
  group, scale = case['heads'] // case['kv_heads'], 1 / math.sqrt(case['dim'])
  out = torch.zeros(q.shape, dtype=torch.float64, device='cuda')
  dq = torch.zeros_like(out)
  dk, dv = (torch.zeros(k.shape, dtype=torch.float64, device='cuda') for _ in range(2))
  step = max(1, 2 ** 27 // case['keys'])
  for b in range(case['batch']):
    index = torch.arange(case['keys'], device='cuda')
    if state['key_lengths'] is not None:
      index = index[:int(state['key_lengths'][b])]
    elif state['key_mask'] is not None:
      index = index[state['key_mask'][b]]
    if len(index) == 0:
      continue
    for h in range(case['heads']):
      kh, vh = k[b, index, h // group].double(), v[b, index, h // group].double()
      for r in range(0, case['queries'], step):
        qh = q[b, r:r + step, h].double()
        p = torch.softmax(scale * (qh @ kh.T), -1)
        out[b, r:r + step, h] = p @ vh
        if case['train']:
          dy = state['dy'][b, r:r + step, h].double()
          dv[b, index, h // group] += p.T @ dy
          ds = p * (dy @ vh.T - (dy * out[b, r:r + step, h]).sum(-1, keepdim=True)) * scale
          dq[b, r:r + step, h] = ds @ kh
          dk[b, index, h // group] += ds.T @ qh
  return [out, dq, dk, dv] if case['train'] else [out]
