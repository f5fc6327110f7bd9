"""A learned readout of a clip's feature grids, as the integration notes write it: TAPIR's backbone gives the tokens, points attend to
them through tapnet_amd.attention, and a training step's gradients agree with plain operations in 64 bits."""
import math

import pytest
import torch

from tests.golden_util import load_case

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, POINTS = 4, 2, 32, 40


class Plain:
  """The operators from their formulas, for autograd in 64 bits."""

  @staticmethod
  def layer_norm(x, w, b):
    c = x - x.mean(-1, keepdim=True)
    return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b

  @staticmethod
  def rotary_positions(x, p):
    parts, begin = [], 0
    for a, width in enumerate([12, 10, 10]):
      i = torch.arange(width // 2, device=x.device)
      angle = (p[..., a, None].double() * 10000.0 ** (-2.0 * i.double() / width)).unsqueeze(-2)
      lo, hi = x[..., begin:begin + width // 2], x[..., begin + width // 2:begin + width]
      parts += [lo * angle.cos() - hi * angle.sin(), lo * angle.sin() + hi * angle.cos()]
      begin += width
    return torch.cat(parts, -1)

  @staticmethod
  def cross_attention(q, k, v, key_lengths):
    k, v = (t.repeat_interleave(HEADS // KV_HEADS, 2).permute(0, 2, 1, 3) for t in (k, v))
    s = q.permute(0, 2, 1, 3) @ k.transpose(2, 3).contiguous() / math.sqrt(DIM)
    gone = torch.arange(k.shape[2], device=q.device) >= key_lengths[:, None].long()
    return (torch.softmax(s.masked_fill(gone[:, None, None], -math.inf), -1) @ v).permute(0, 2, 1, 3)


def readout(ops, tokens, points, w, b, wq, wkv, at_points, at_cells, cells_of_each_clip):
  batch, n = points.shape[:2]
  x, t = ops.layer_norm(points, w, b), ops.layer_norm(tokens, w, b)
  q = (x @ wq).view(batch, n, HEADS, DIM)
  k, v = (t @ wkv).view(batch, -1, 2, KV_HEADS, DIM).unbind(2)
  q, k = ops.rotary_positions(q, at_points), ops.rotary_positions(k, at_cells)
  return ops.cross_attention(q, k, v, key_lengths=cells_of_each_clip)


@pytest.fixture(scope='module')
def clip():
  """Tokens of two clips: a golden clip's grid, and the same of which the last frames are missing."""
  from tapnet_amd import tapir_model
  cfg, g, weights = load_case('tapir')
  model = tapir_model.TAPIR(pyramid_level=cfg['pyramid_level'], extra_convs=cfg['extra_convs'], softmax_temperature=cfg['softmax_temperature'],
                            initial_resolution=(cfg['res'], cfg['res']), weights=weights, device='cuda:0')
  grid = torch.as_tensor(model.get_feature_grids(g['video']).lowres[0]).cuda()
  _, frames, h, w, _ = grid.shape
  cells = torch.stack(torch.meshgrid(*(torch.arange(float(n), device='cuda') for n in (frames, h, w)), indexing='ij'), -1).flatten(0, 2)
  lengths = torch.tensor([frames * h * w, (frames // 2) * h * w], dtype=torch.int32, device='cuda')
  return grid.flatten(1, 3).expand(2, -1, -1).contiguous(), cells, lengths


def leaves_of(tokens, cells, dtype):
  gen = torch.Generator(device='cuda').manual_seed(5)
  randn = lambda *shape: torch.randn(*shape, generator=gen, device='cuda')
  c = tokens.shape[-1]
  at = cells.amax(0) * torch.rand(2, POINTS, 3, generator=gen, device='cuda')
  leaves = [tokens.to(dtype), randn(2, POINTS, c).to(dtype), 1 + 0.1 * randn(c), 0.1 * randn(c),
            (randn(c, HEADS * DIM) / math.sqrt(c)).to(dtype), (randn(c, 2 * KV_HEADS * DIM) / math.sqrt(c)).to(dtype)]
  return [t.detach().requires_grad_() for t in leaves], at, randn(2, POINTS, HEADS, DIM).to(dtype)


def test_training_step_on_feature_grids(clip):
  """f32.  Each step's relative error is some hundred u at most; six steps in a row, amplified by the softmax by at most the
  scores' size (below 20 here), stay below 1e-4 of the largest value."""
  from tapnet_amd import attention
  tokens, cells, lengths = clip
  leaves, at, dout = leaves_of(tokens, cells, torch.float32)
  y = readout(attention, *leaves, at, cells, lengths)
  grads = torch.autograd.grad(y, leaves, dout)
  plain = [t.detach().double().requires_grad_() for t in leaves]
  want = readout(Plain, *plain, at, cells, lengths)
  want_grads = torch.autograd.grad(want, plain, dout.double())
  for got, ref in zip((y, *grads), (want, *want_grads)):
    assert float((got.detach().double() - ref.detach()).abs().max()) <= 1e-4 * float(ref.detach().abs().max())
  assert (grads[0][1, int(lengths[1]):] == 0).all()     # the cells that the second clip does not have


def test_training_step_on_feature_grids_in_bf16(clip):
  """The same step in bf16 runs, gives every leaf a finite gradient of its type and the same bits twice."""
  from tapnet_amd import attention
  tokens, cells, lengths = clip
  leaves, at, dout = leaves_of(tokens, cells, torch.bfloat16)
  first, again = ([y.detach(), *torch.autograd.grad(y, leaves, dout)]
                  for y in (readout(attention, *leaves, at, cells, lengths) for _ in range(2)))
  for t, leaf in zip(first[1:], leaves):
    assert t.dtype == leaf.dtype and t.shape == leaf.shape and torch.isfinite(t.float()).all() and bool(t.any())
  assert torch.equal(first[0], again[0]) and all(torch.equal(a, b) for a, b in zip(first[1:4], again[1:4]))
