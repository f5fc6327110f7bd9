"""Recorded programs of tapnet_amd.attention's operators, replayed on an MI355X with other inputs, against the eager calls."""
import pytest
import torch
from torch._subclasses import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from tests import test_gpu_attention as T

pytestmark = pytest.mark.gpu

DTYPES, IDS = T.DTYPES, T.IDS
A = T.A


def program(A, lengths, at):
  def fn(q, k, v, weight, bias):
    return A.cross_attention(A.rotary_positions(A.layer_norm(q, weight, bias), at, base=(100.0, 50.0)), k, v, key_lengths=lengths)
  return fn


def inputs_of(seed, dtype):
  gen = T.generator(seed)
  (q, k, v), dout = T.attention_inputs(gen, dtype, 2, 37, 300, 4, 2, 32)
  return [t.detach() for t in (q, k, v)] + [1 + 0.1 * T.randn(gen, 32), 0.1 * T.randn(gen, 32)], dout


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_replayed_recordings(A, dtype):
  gen = T.generator(3)
  lengths = torch.tensor([300, 77], dtype=torch.int32, device='cuda')
  fn = program(A, lengths, torch.rand(37, 2, generator=gen, device='cuda') * 50)
  first, dout = inputs_of(1, dtype)

  def step(*tensors):
    leaves = [t.detach().requires_grad_() for t in tensors[:-1]]
    y = fn(*leaves)
    return [y.detach(), *torch.autograd.grad(y, leaves, tensors[-1])]
  traced = torch.jit.trace(fn, tuple(first))
  forward, training = make_fx(fn)(*first), make_fx(step)(*first, dout)
  for seed in (2, 3):
    other, dout = inputs_of(seed, dtype)
    want = step(*other, dout)
    assert torch.equal(forward(*other), want[0])
    assert all(torch.equal(a, b) for a, b in zip(training(*other, dout), want))
    leaves = [t.requires_grad_() for t in other]
    y = traced(*leaves)
    assert torch.equal(y, want[0])
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dout), want[1:]))


def test_under_dispatch_modes(A):
  """Shapes without memory, and a mode that only looks on."""
  first, dout = inputs_of(1, torch.bfloat16)
  lengths, at = torch.tensor([300, 77], dtype=torch.int32, device='cuda'), torch.zeros(37, 2, device='cuda')
  want = program(A, lengths, at)(*first)
  with FlopCounterMode(display=False):
    assert torch.equal(program(A, lengths, at)(*first), want)
  with FakeTensorMode() as mode:
    fake = [mode.from_tensor(t).requires_grad_() for t in first]
    y = program(A, mode.from_tensor(lengths), mode.from_tensor(at))(*fake)
    assert y.shape == want.shape and y.dtype == want.dtype and y.device == want.device
    for g, t in zip(torch.autograd.grad(y, fake, mode.from_tensor(dout)), fake):
      assert g.shape == t.shape and g.dtype == t.dtype


def test_checkpointed(A):
  """Recomputed in the backward pass: the same bits."""
  from torch.utils.checkpoint import checkpoint
  first, dout = inputs_of(4, torch.float32)
  leaves = [t.requires_grad_() for t in first]
  fn = program(A, torch.tensor([300, 0], dtype=torch.int32, device='cuda'), torch.zeros(37, 2, device='cuda'))
  want = torch.autograd.grad(fn(*leaves), leaves, dout)
  got = torch.autograd.grad(checkpoint(fn, *leaves, use_reentrant=False), leaves, dout)
  assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('name', ['layer_norm', 'rotary_positions', 'cross_attention'])
def test_a_backward_pass_captured_over_a_live_eager_graph_is_refused(A, name):
  """An error of the call, not the end of the process; without the eager graph the same capture works."""
  gen = T.generator(9)
  x = T.randn(gen, 1, 6, 2, 32).requires_grad_()
  k, at, dy = T.randn(gen, 1, 9, 2, 32), torch.rand(6, 2, generator=gen, device='cuda'), T.randn(gen, 1, 6, 2, 32)
  fn = {'layer_norm': lambda: A.layer_norm(x), 'rotary_positions': lambda: A.rotary_positions(x, at),
        'cross_attention': lambda: A.cross_attention(x, k, k)}[name]
  step = lambda: torch.autograd.grad(fn(), [x], dy)[0]
  want = step()
  alive = fn()
  print('capture over a live eager graph', flush=True)
  with pytest.raises(RuntimeError, match='eager autograd graph'):
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
      step()
  torch.cuda.synchronize()
  del alive
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = step()
  for _ in range(3):
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
