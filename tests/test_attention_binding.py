"""The operators of tapnet_amd.attention as torch's dispatcher has them: recorded programs hold them, shapes without memory, what is
refused.  Tensors are on torch's meta device here; tests/test_gpu_attention_binding.py replays recordings on the GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from tapnet_amd import attention as A

DTYPES = [torch.float32, torch.bfloat16]
IDS = ['f32', 'bf16']


def meta(*shape, dtype=torch.float32):
  return torch.empty(*shape, dtype=dtype, device='meta')


def calls(dtype):
  """(function, tensors it differentiates) of every operator."""
  f = lambda *shape: meta(*shape, dtype=dtype)
  positions, lengths, mask = meta(5, 3), torch.empty(2, dtype=torch.int32, device='meta'), torch.empty(2, 7, dtype=torch.bool, device='meta')
  return {
      'layer_norm': (lambda x, w, b: A.layer_norm(x, w, b), [f(2, 5, 24), meta(24), meta(24)]),
      'rotary_positions': (lambda x: A.rotary_positions(x, positions), [f(2, 5, 4, 24)]),
      'cross_attention': (lambda q, k, v: A.cross_attention(q, k, v, lengths, mask), [f(2, 5, 4, 24), f(2, 7, 2, 24), f(2, 7, 2, 24)]),
  }


NAMES = ['layer_norm', 'rotary_positions', 'cross_attention']


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('name', NAMES)
def test_shapes_and_types(name, dtype):
  fn, inputs = calls(dtype)[name]
  y = fn(*inputs)
  assert y.shape == inputs[0].shape and y.dtype == dtype and not y.requires_grad
  inputs = [t.requires_grad_() for t in inputs]
  y = fn(*inputs)
  assert y.requires_grad
  for g, t in zip(torch.autograd.grad(y, inputs, torch.empty_like(y)), inputs):
    assert g.shape == t.shape and g.dtype == t.dtype
  (g,) = torch.autograd.grad(fn(*inputs), inputs[-1:], torch.empty_like(y))
  assert g.shape == inputs[-1].shape


@pytest.mark.parametrize('name', NAMES)
def test_recordings_hold_the_operators(name):
  fn, inputs = calls(torch.float32)[name]
  traced = torch.jit.trace(fn, tuple(inputs), check_trace=False)
  kinds = [n.kind() for n in traced.graph.nodes()]
  assert 'tapnet_amd::' + name in kinds and 'aten::empty' not in kinds, kinds

  def step(*tensors):
    tensors = [t.detach().requires_grad_() for t in tensors]
    y = fn(*tensors)
    return [y, *torch.autograd.grad(y, tensors, torch.ones_like(y))]
  for program, wanted in ((fn, 1), (step, 2)):
    graph = make_fx(program)(*inputs)
    targets = [str(n.target) for n in graph.graph.nodes if n.op == 'call_function']
    assert sum(t.startswith('tapnet_amd.' + name) for t in targets) == wanted, targets
    assert not any('empty' in t for t in targets), targets


@pytest.mark.parametrize('name', NAMES)
def test_tangents_are_refused(name):
  """A tangent would be dropped: whichever tensor has it, with and without gradients."""
  fn, inputs = calls(torch.float32)[name]
  with fwd.dual_level():
    for n in range(len(inputs)):
      for grad in (False, True):
        dual = [t.detach().requires_grad_(grad) for t in inputs]
        dual[n] = fwd.make_dual(dual[n], torch.empty_like(dual[n]))
        with pytest.raises(RuntimeError, match='forward-mode'):
          fn(*dual)
    positions = fwd.make_dual(meta(5, 3), meta(5, 3))
    with pytest.raises(RuntimeError, match='forward-mode'):
      A.rotary_positions(meta(2, 5, 4, 24), positions)


def test_operators_below_autograd_check_what_they_get():
  """A recording is a program that can be called with other tensors."""
  ops = torch.ops.tapnet_amd
  A._ops()
  x, stats = meta(5, 24), meta(2, 5)
  ops.layer_norm_backward(x, None, stats, x, True, True, False)
  for bad in ((x, None, meta(2, 4), x, True, False, False), (x, None, stats, meta(4, 24), True, False, False),
              (x, None, stats, x.bfloat16(), True, False, False), (x, meta(23), stats, x, True, False, False),
              (x, None, stats.bfloat16(), x, True, False, False)):
    with pytest.raises(ValueError):
      ops.layer_norm_backward(*bad)
  q, k, lengths = meta(2, 3, 4, 16), meta(2, 7, 2, 16), torch.empty(2, dtype=torch.int32, device='meta')
  good = dict(q=q, k=k, v=k, key_lengths=lengths, key_mask=None, scale=0.5, out_f32=q, stats=meta(2, 12, 2), dout=q, want_q=True, want_kv=True)
  assert [t.shape for t in ops.cross_attention_backward(**good)] == [q.shape, k.shape, k.shape]
  for bad in (dict(dout=meta(2, 3, 4, 8)), dict(out_f32=meta(2, 3, 2, 16)), dict(stats=meta(2, 11, 2)), dict(v=meta(2, 7, 2, 8)),
              dict(key_lengths=lengths[:1]), dict(scale=-1.0), dict(dout=q.bfloat16()), dict(out_f32=q.bfloat16())):
    with pytest.raises(ValueError):
      ops.cross_attention_backward(**{**good, **bad})
  with pytest.raises(ValueError):
    ops.rotary_positions_turn(q, meta(3, 2), [8, 10], [10000.0], False, True)
  with pytest.raises(ValueError):
    ops.rotary_positions_turn(q, meta(3, 2), [8, 8], [1.0, 2.0, 3.0], False, True)


def test_cpu_tensors_are_refused():
  q, k = torch.zeros(1, 2, 2, 8), torch.zeros(1, 3, 2, 8)
  for call in (lambda: A.layer_norm(q), lambda: A.rotary_positions(q, torch.zeros(2, 1)), lambda: A.cross_attention(q, k, k),
               lambda: A.layer_norm(q.requires_grad_()), lambda: A.cross_attention(q.requires_grad_(), k, k)):
    with pytest.raises(ValueError, match='GPU'):
      call()


def test_scales_out_of_range_are_refused():
  q = meta(1, 2, 2, 8)
  for scale in (1.2e-38, 2.0 ** -61, 2.0 ** 61, 3e38, 1e39, float('nan'), float('inf')):
    with pytest.raises(ValueError, match='scale'):
      A.cross_attention(q, q, q, scale=scale)
  for scale in (2.0 ** -60, 2.0 ** 60):
    A.cross_attention(q, q, q, scale=scale)


def test_layer_norm_channels_past_32_bits_are_refused():
  with pytest.raises(ValueError, match='channels'):
    A.layer_norm(meta(2 ** 30 + 1))
  assert A.layer_norm(meta(2 ** 30)).shape == (2 ** 30,)
