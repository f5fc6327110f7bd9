"""tapnet_amd.attention on an MI355X: layer normalisation, rotary positions and cross attention with their gradients against
64-bit forms with counted roundings (tests/attention_ref.py), at lengths from one token to a clip's, on strided and padded
batches, on side streams, from two threads and in captured graphs, alone and one after the other as a readout uses them."""
import math
import threading

import pytest
import torch

from tests import attention_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
IDS = ['f32', 'bf16']


@pytest.fixture(scope='module')
def A():
  from tapnet_amd import attention
  return attention


def generator(seed):
  return torch.Generator(device='cuda').manual_seed(seed)


def randn(gen, *shape):
  return torch.randn(*shape, generator=gen, device='cuda')


def grads_of(y, inputs, dy):
  return torch.autograd.grad(y, inputs, dy)


# ------------------------------------------------------------------------------------------------------ layer norm
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('shape,affine,pad', [
    ((1, 1), 'full', 0), ((7, 13), 'full', 0), ((2, 3, 64), 'scale', 0), ((1024, 256), 'full', 0), ((5, 1000), 'none', 8),
    ((3001, 257), 'full', 0), ((2, 48, 512), 'scale', 16), ((4097, 128), 'full', 0), ((9, 2048), 'bias', 0), ((11, 4096), 'full', 0),
    ((3, 20001), 'full', 0), ((0, 32), 'full', 0)])
def test_layer_norm(A, dtype, shape, affine, pad):
  gen = generator(shape[-1] + shape[0])
  n = shape[-1]
  x = (2 * randn(gen, *shape[:-1], n + pad) + 3 * randn(gen, *shape[:-1], 1)).to(dtype)[..., :n].requires_grad_()
  weight = (1 + 0.3 * randn(gen, n)).requires_grad_() if affine in ('full', 'scale') else None
  bias = (0.3 * randn(gen, n)).requires_grad_() if affine in ('full', 'bias') else None
  dy = randn(gen, *shape).to(dtype)
  y = A.layer_norm(x, weight, bias)
  inputs = [t for t in (x, weight, bias) if t is not None]
  got = iter(grads_of(y, inputs, dy))
  with torch.no_grad():
    want = R.layer_norm(x, weight, bias, 1e-5, dy)
    R.check('y', y, want[0])
    for name, w in zip(('dx', 'dweight', 'dbias'), want[1:]):
      if w is not None:
        R.check(name, next(got), w)
    assert torch.equal(A.layer_norm(x, weight, bias), y.detach())


def test_layer_norm_gradients_of_some_inputs(A):
  """Parameters alone, the input alone, a gradient that is a broadcast number, permuted axes."""
  gen = generator(3)
  x = randn(gen, 6, 5, 40)
  weight, bias = (1 + 0.3 * randn(gen, 40)).requires_grad_(), torch.zeros(40, device='cuda')
  (dw,) = grads_of(A.layer_norm(x, weight, bias).sum(), [weight], None)
  ones = torch.ones_like(x)
  R.check('dweight', dw, R.layer_norm(x, weight.detach(), bias, 1e-5, ones)[2])
  xt = x.permute(1, 0, 2).detach().requires_grad_()
  y = A.layer_norm(xt, weight.detach())
  (dx,) = grads_of(y.sum(), [xt], None)
  want = R.layer_norm(xt.detach(), weight.detach(), None, 1e-5, ones.permute(1, 0, 2))
  R.check('y', y.detach(), want[0])
  R.check('dx', dx, want[1])


def test_layer_norm_matches_the_engines_own(A):
  """The norm of the ExtraConvs path (tapir_layernorm_affine) and this one are the same function of the same rows."""
  import ctypes
  from tapnet_amd import _ffi
  gen = generator(8)
  x, weight, bias = randn(gen, 777, 256), 1 + 0.2 * randn(gen, 256), 0.2 * randn(gen, 256)
  y = A.layer_norm(x, weight, bias)
  lib, other = _ffi.load_library(), torch.empty_like(x)
  ctx, cfg = ctypes.c_void_p(), _ffi.TapirCfg(1, 4, 12, 0, 20.0, 256, 256, _ffi.TAPIR_F32)
  assert lib.tapir_create(ctypes.byref(ctx), ctypes.byref(cfg), x.device.index) == 0
  rc = lib.tapir_layernorm_affine(ctx, x.data_ptr(), weight.data_ptr(), bias.data_ptr(), other.data_ptr(), 777, 256,
                                  torch.cuda.current_stream().cuda_stream)
  torch.cuda.synchronize()
  lib.tapir_destroy(ctx)
  assert rc == 0
  value, bound = R.layer_norm(x, weight, bias, 1e-5)[0]
  R.check('this', y, (value, bound))
  R.check('the other', other, (value, bound))


# ------------------------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('interleaved', [False, True], ids=['halves', 'pairs'])
@pytest.mark.parametrize('batch,tokens,heads,dim,sections,shared', [
    (1, 1, 1, 2, None, False), (2, 257, 4, 64, None, True), (1, 4097, 8, 32, [8, 12, 12], False), (3, 100, 6, 40, None, False),
    (1, 33, 3, 7, [2, 2, 2], False), (1, 2048, 2, 128, [64, 32, 32], True), (2, 19, 1, 256, [100, 0, 96], False),
    (2, 0, 4, 64, None, False)])
def test_rotary_positions(A, dtype, interleaved, batch, tokens, heads, dim, sections, shared):
  gen = generator(dim + tokens)
  x = randn(gen, batch, tokens, heads, dim).to(dtype).requires_grad_()
  axes = 1 if dim == 2 else len(sections) if sections else 3
  positions = torch.rand(*(() if shared else (batch,)), tokens, axes, generator=gen, device='cuda') * 512 - 10
  y = A.rotary_positions(x, positions, sections, base=10000.0, interleaved=interleaved)
  if sections is None:
    pairs = dim // 2
    sections = [2 * (pairs // axes + (a < pairs % axes)) for a in range(axes)]
  dy = randn(gen, batch, tokens, heads, dim).to(dtype)
  (dx,) = grads_of(y, [x], dy)
  bases = [10000.0] * axes
  R.check('y', y.detach(), R.rotary(x.detach(), positions, sections, bases, interleaved))
  R.check('dx', dx, R.rotary(dy, positions, sections, bases, interleaved, inverse=True))


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_rotary_positions_strides_and_far_positions(A, dtype):
  """Heads-first tensors, a slice of a fused projection, channels apart, an expanded gradient; frames far into a video."""
  gen = generator(1)
  positions = torch.tensor([[0.0, 0.5], [99999.0, -3.25], [1e6 + 0.5, 2.0 ** 24], [1e-30, 7.0]], device='cuda')
  fused = randn(gen, 2, 4, 3, 5, 48).to(dtype)
  for x in (fused[:, :, 1], fused[:, :, 2].transpose(2, 3).contiguous().transpose(2, 3), fused[:, :, 0].transpose(1, 2).contiguous().transpose(1, 2),
            fused[:, :, 1, :, 1:41]):
    sections = [x.shape[-1] // 2] * 2
    x = x.detach().requires_grad_()
    y = A.rotary_positions(x, positions, sections, base=(10000.0, 50.0))
    (dx,) = grads_of(y.sum(), [x], None)
    R.check('y', y.detach(), R.rotary(x.detach(), positions, sections, [10000.0, 50.0], False))
    R.check('dx', dx, R.rotary(torch.ones_like(y), positions, sections, [10000.0, 50.0], False, inverse=True))


# ------------------------------------------------------------------------------------------------- cross attention
def attention_inputs(gen, dtype, batch, queries, keys, heads, kv_heads, dim, packed=True):
  q = randn(gen, batch, queries, heads, dim)
  if packed:
    k, v = randn(gen, batch, keys, 2, kv_heads, dim).to(dtype).unbind(2)
  else:
    k, v = randn(gen, batch, keys, kv_heads, dim).to(dtype), randn(gen, batch, keys, kv_heads, dim).to(dtype)
  if keys:
    like = k[:, torch.randint(0, keys, (queries,), generator=gen, device='cuda')].float().repeat_interleave(heads // kv_heads, 2)
    q[:, ::2] = 0.5 * q[:, ::2] + like[:, ::2]
  return [t.detach().requires_grad_() for t in (q.to(dtype), k, v)], randn(gen, batch, queries, heads, dim).to(dtype)


def check_attention(A, inputs, dout, lengths=None, mask=None, scale=None):
  q, k, v = inputs
  keep = torch.ones(k.shape[:2], dtype=torch.bool, device='cuda') if mask is None else mask.clone()
  if lengths is not None:
    keep &= torch.arange(k.shape[1], device='cuda') < lengths[:, None].long()
  out = A.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask, scale=scale)
  grads = grads_of(out, [q, k, v], dout)
  with torch.no_grad():
    want = R.attention(q, k, v, keep, q.shape[-1] ** -0.5 if scale is None else scale, dout)
    for name, g, w in zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *grads), want):
      assert g.dtype == q.dtype
      R.check(name, g, w)
    # the same call without gradients gives the same bits, and so does the same call again
    assert torch.equal(A.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask, scale=scale), out)
  again = grads_of(A.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask, scale=scale), [q, k, v], dout)
  assert all(torch.equal(a, b) for a, b in zip(again, grads))
  return out.detach(), grads


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('batch,queries,keys,heads,kv_heads,dim', [
    (1, 1, 1, 1, 1, 8), (1, 1, 4099, 8, 2, 64), (2, 3, 33, 4, 4, 32), (1, 257, 1024, 8, 8, 32), (1, 31, 3000, 4, 1, 128),
    (3, 129, 65, 6, 2, 96), (1, 2, 20000, 4, 4, 64), (1, 2000, 17, 4, 2, 40), (1, 700, 1900, 2, 2, 64), (2, 5, 0, 2, 2, 32),
    (2, 0, 7, 2, 1, 32), (1, 64, 64, 1, 1, 120), (2, 200, 700, 4, 2, 72), (1, 65, 130, 2, 1, 88), (1, 9, 3000, 8, 2, 96), (2, 520, 40, 4, 1, 104)])
def test_cross_attention(A, dtype, batch, queries, keys, heads, kv_heads, dim):
  gen = generator(queries * 7 + keys)
  inputs, dout = attention_inputs(gen, dtype, batch, queries, keys, heads, kv_heads, dim)
  check_attention(A, inputs, dout)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('how', ['lengths', 'mask', 'both'])
@pytest.mark.parametrize('queries,keys', [(1, 700), (150, 333), (3, 5000)])
def test_cross_attention_masks(A, dtype, how, queries, keys):
  """Padding that holds NaN and infinities, clips without a token, lengths out of range, a mask that leaves nothing."""
  batch, heads, kv_heads, dim = 5, 4, 2, 64
  gen = generator(keys)
  inputs, dout = attention_inputs(gen, dtype, batch, queries, keys, heads, kv_heads, dim)
  lengths = torch.tensor([keys, keys // 2 + 1, 0, -4, keys + 1000], dtype=torch.int32, device='cuda') if how != 'mask' else None
  mask = torch.rand(batch, keys, generator=gen, device='cuda') < 0.6 if how != 'lengths' else None
  if mask is not None:
    mask[1] = False
    mask[0, :130] = False
  keep = torch.ones(batch, keys, dtype=torch.bool, device='cuda') if mask is None else mask.clone()
  if lengths is not None:
    keep &= torch.arange(keys, device='cuda') < lengths[:, None].long()
  bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max, torch.finfo(dtype).min], device='cuda')
  gone = (~keep).nonzero()
  for t in inputs[1:]:
    t.data[gone[:, 0], gone[:, 1]] = bad[torch.randint(0, 5, (len(gone), 1, 1), generator=gen, device='cuda')].to(dtype)
  out, grads = check_attention(A, inputs, dout, lengths, mask)
  empty = ~keep.any(1)
  assert empty.any() and (out[empty] == 0).all() and (grads[0][empty] == 0).all()
  assert (grads[1][~keep] == 0).all() and (grads[2][~keep] == 0).all()


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_cross_attention_strides(A, dtype):
  """Heads-first tensors, rows at odd addresses and channels apart (both copied), broadcast keys, an expanded gradient."""
  gen = generator(4)
  (q, k, v), dout = attention_inputs(gen, dtype, 2, 37, 90, 4, 2, 32, packed=False)
  heads_first = [t.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for t in (q, k, v)]
  check_attention(A, heads_first, dout)
  odd = [torch.empty(*t.shape[:3], t.shape[3] + 3, dtype=dtype, device='cuda')[..., 1:33].copy_(t.detach()).detach().requires_grad_()
         for t in (q, k, v)]
  check_attention(A, odd, dout)
  apart = [t.detach().transpose(2, 3).contiguous().transpose(2, 3).requires_grad_() for t in (q, k, v)]
  check_attention(A, apart, dout)
  one = k.detach()[:1].clone().requires_grad_()
  out = A.cross_attention(q, one.expand(2, -1, -1, -1), v)
  dq, done, dv = grads_of(out.sum(), [q, one, v], None)
  want = R.attention(q.detach(), one.detach().expand(2, -1, -1, -1), v.detach(), torch.ones(2, 90, dtype=torch.bool, device='cuda'),
                     32 ** -0.5, torch.ones_like(dout))
  R.check('dq', dq, want[1])
  value, bound = want[2][0].sum(0, keepdim=True), want[2][1].sum(0, keepdim=True)
  R.check('dk of a broadcast', done, (value, bound + R.unit(dtype) * (value.abs() + bound)))
  R.check('dv', dv, want[3])


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('batch,queries,keys', [(70, 3, 300), (70, 400, 200), (9, 70, 1500)])
def test_cross_attention_many_clips(A, dtype, batch, queries, keys):
  """More clips than a wave has lanes, of all lengths from none to whole."""
  gen = generator(13)
  inputs, dout = attention_inputs(gen, dtype, batch, queries, keys, 2, 1, 32)
  lengths = torch.randint(0, keys + 1, (batch,), generator=gen, device='cuda').to(torch.int32)
  lengths[0], lengths[1], lengths[-1], lengths[-2] = 0, keys, keys, 0
  check_attention(A, inputs, dout, lengths)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_gradients_of_some_inputs(A, dtype):
  """Only what is asked for is computed, with the bits of the whole backward pass; no second derivative."""
  gen = generator(14)
  inputs, dout = attention_inputs(gen, dtype, 2, 40, 300, 4, 2, 64)
  lengths = torch.tensor([300, 11], dtype=torch.int32, device='cuda')
  whole = grads_of(A.cross_attention(*inputs, key_lengths=lengths), inputs, dout)
  for wanted in ([0], [1], [2], [0, 2], [1, 2]):
    some = [t if n in wanted else t.detach() for n, t in enumerate(inputs)]
    for args in (some, inputs):       # the others need no gradient, or none is asked for
      got = grads_of(A.cross_attention(*args, key_lengths=lengths), [inputs[n] for n in wanted], dout)
      assert all(torch.equal(g, whole[n]) for g, n in zip(got, wanted))
  x = randn(gen, 5, 7, 32).to(dtype).requires_grad_()
  weight, bias = randn(gen, 32).requires_grad_(), randn(gen, 32).requires_grad_()
  all_of = grads_of(A.layer_norm(x, weight, bias).sum(), [x, weight, bias], None)
  for n, t in enumerate((x, weight, bias)):
    assert torch.equal(grads_of(A.layer_norm(x, weight, bias).sum(), [t], None)[0], all_of[n])
  assert torch.equal(grads_of(A.layer_norm(x, None, bias).sum(), [bias], None)[0], all_of[2])
  positions = torch.rand(40, 3, generator=gen, device='cuda')
  for y, leaf in ((A.cross_attention(*inputs), inputs[0]), (A.layer_norm(x, weight, bias), x), (A.layer_norm(x), x),
                  (A.rotary_positions(inputs[0], positions), inputs[0])):
    (g,) = torch.autograd.grad(y.float().square().sum(), [leaf], create_graph=True, retain_graph=True)
    with pytest.raises(RuntimeError, match='second derivative'):
      g.sum().backward()
    (g,) = torch.autograd.grad(y.float().square().sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError):
      torch.autograd.grad(g.sum(), [leaf])


def test_rows_far_apart(A):
  """Tokens 2^22 elements and more apart: copied; a single token's stride does not matter."""
  gen = generator(16)
  (q, k, v), dout = attention_inputs(gen, torch.bfloat16, 1, 3, 5, 2, 2, 32, packed=False)
  far = torch.zeros(5, 1 << 22, dtype=torch.bfloat16, device='cuda')[:, :64].view(1, 5, 2, 32)
  far.copy_(k.detach())
  assert far.stride(1) == 1 << 22
  assert torch.equal(A.cross_attention(q, far, v), A.cross_attention(q, k, v))


def test_cross_attention_gradient_against_differences(A):
  """Central differences of the float32 forward pass along random directions: the truncation is third order in the step, the
  outputs' own error (their bound) is divided by it."""
  gen = generator(12)
  inputs, dout = attention_inputs(gen, torch.float32, 1, 20, 50, 2, 1, 16)
  grads = grads_of(A.cross_attention(*inputs), inputs, dout)
  keep = torch.ones(1, 50, dtype=torch.bool, device='cuda')
  step = 2.0 ** -6
  for n, t in enumerate(inputs):
    direction = randn(gen, *t.shape) / math.sqrt(t.numel())

    def value(s):
      moved = [u.detach() + (s * direction if m == n else 0) for m, u in enumerate(inputs)]
      y = A.cross_attention(*moved).double()
      return (y * dout.double()).sum(), R.attention(*moved, keep, 0.25)[0]
    (hi, (_, e_hi)), (lo, (_, e_lo)), (hi2, _), (lo2, _) = value(step), value(-step), value(step / 2), value(-step / 2)
    coarse, fine = (hi - lo) / (2 * step), (hi2 - lo2) / step
    got = (grads[n].double() * direction.double()).sum()
    noise = ((e_hi + e_lo) * dout.double().abs()).sum() / step * 2
    moved_rounding = 2.0 ** -24 * (t.detach().double().abs() * grads[n].double().abs()).sum() / step * 2
    # Richardson: the error of the extrapolated difference is below the change the refinement made
    extrapolated = fine + (fine - coarse) / 3
    assert abs(got - extrapolated) <= abs(fine - coarse) + noise + moved_rounding, (n, float(got), float(extrapolated))


# --------------------------------------------------------------------------------------- streams, threads, graphs, order
def readout(A, points, tokens, weight, bias, wq, wkv, at_points, at_tokens, lengths):
  """Points read a clip: norm, projections, rotary positions, attention."""
  batch, n, c = points.shape
  heads, dim = 4, 32
  x, t = A.layer_norm(points, weight, bias), A.layer_norm(tokens, weight, bias)
  q = (x @ wq).view(batch, n, heads, dim)
  k, v = (t @ wkv).view(batch, tokens.shape[1], 2, 2, dim).unbind(2)
  q, k = A.rotary_positions(q, at_points), A.rotary_positions(k, at_tokens)
  return A.cross_attention(q, k, v, key_lengths=lengths)


def readout_inputs(gen, dtype):
  batch, n, m, c = 2, 50, 600, 128
  leaves = [randn(gen, batch, n, c).to(dtype), randn(gen, batch, m, c).to(dtype), 1 + 0.1 * randn(gen, c), 0.1 * randn(gen, c),
            (randn(gen, c, 128) / math.sqrt(c)).to(dtype), (randn(gen, c, 128) / math.sqrt(c)).to(dtype)]
  leaves = [t.requires_grad_() for t in leaves]
  at = [torch.rand(batch, n, 3, generator=gen, device='cuda') * 48, torch.rand(m, 3, generator=gen, device='cuda') * 48]
  return leaves, at, torch.tensor([600, 333], dtype=torch.int32, device='cuda'), randn(gen, batch, n, 4, 32).to(dtype)


def test_readout_f32_against_autograd_in_64_bits(A):
  """The operators together, forward and backward, against torch's autograd on plain float64 operations.  Each step's relative
  error is some hundred u at most (its bound in attention_ref.py for these sizes); six steps in a row, amplified by the softmax
  by at most the scores' size (below 20 here), stay below 1e-4 of the largest value."""
  gen = generator(21)
  leaves, at, lengths, dout = readout_inputs(gen, torch.float32)
  out = readout(A, *leaves, *at, lengths)
  grads = grads_of(out, leaves, dout)

  class Plain:
    @staticmethod
    def layer_norm(x, w, b):
      c = x - x.mean(-1, keepdim=True)
      return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b

    @staticmethod
    def rotary_positions(x, p):
      parts, begin = [], 0
      for a, width in enumerate([12, 10, 10]):
        i = torch.arange(width // 2, device='cuda')
        angle = (p[..., a, None].double() * 10000.0 ** (-2.0 * i.double() / width)).unsqueeze(-2)
        lo, hi = x[..., begin:begin + width // 2], x[..., begin + width // 2:begin + width]
        parts += [lo * angle.cos() - hi * angle.sin(), lo * angle.sin() + hi * angle.cos()]
        begin += width
      return torch.cat(parts, -1)

    @staticmethod
    def cross_attention(q, k, v, key_lengths):
      k, v = (t.repeat_interleave(2, 2).permute(0, 2, 1, 3) for t in (k, v))
      s = q.permute(0, 2, 1, 3) @ k.transpose(2, 3).contiguous() / math.sqrt(32)
      gone = torch.arange(k.shape[2], device='cuda') >= key_lengths[:, None].long()
      return (torch.softmax(s.masked_fill(gone[:, None, None], -math.inf), -1) @ v).permute(0, 2, 1, 3)
  plain = [t.detach().double().requires_grad_() for t in leaves]
  want = readout(Plain, *plain, *at, lengths)
  want_grads = grads_of(want, plain, dout.double())
  for g, w in zip((out, *grads), (want, *want_grads)):
    assert float((g.double() - w).abs().max()) <= 1e-4 * float(w.abs().max())


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_side_streams_and_threads(A, dtype):
  """Several readouts at once on streams and threads of their own give the bits of one after the other."""
  gens = [generator(s) for s in (31, 32, 33)]
  cases = [readout_inputs(g, dtype) for g in gens]
  step = lambda leaves, at, lengths, dout: [(o := readout(A, *leaves, *at, lengths)).detach(), *grads_of(o, leaves, dout)]
  want = [step(*c) for c in cases]
  torch.cuda.synchronize()
  got = [None] * len(cases)

  def work(n):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
      for _ in range(5):
        got[n] = step(*cases[n])
    stream.synchronize()
  threads = [threading.Thread(target=work, args=(n,)) for n in range(len(cases))]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  for g, w in zip(got, want):
    assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_captured_graphs(A, dtype):
  """Forward and backward of the operators in two graphs, replayed in turn on new inputs with eager work between them."""
  graphs = []
  for seed in (41, 42):
    gen = generator(seed)
    (q, k, v), dout = attention_inputs(gen, dtype, 2, 5, 3000, 4, 2, 64)
    weight = (1 + 0.1 * randn(gen, 64)).requires_grad_()
    positions = torch.rand(5, 3, generator=gen, device='cuda') * 100
    lengths = torch.tensor([3000, 1], dtype=torch.int32, device='cuda')

    def step(q=q, k=k, v=v, weight=weight, positions=positions, lengths=lengths, dout=dout):
      x = A.rotary_positions(A.layer_norm(q, weight), positions)
      out = A.cross_attention(x, k, v, key_lengths=lengths)
      return [out, *grads_of(out, [q, k, v, weight], dout)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
      step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      results = step()
    graphs.append((graph, results, step, (q, k, v, weight), lengths, gen))
  for turn in range(4):
    for graph, results, step, leaves, lengths, gen in graphs:
      with torch.no_grad():
        for t in leaves:
          t.copy_(randn(gen, *t.shape).to(t.dtype))
        lengths.copy_(torch.tensor([3000 - 700 * turn, 17 * turn], dtype=torch.int32))
      want = step()
      graph.replay()
      torch.cuda.synchronize()
      assert all(torch.equal(a, b) for a, b in zip(results, want)), turn


def test_results_are_written_whole_and_nothing_else(A):
  """Memory around dense results stays as it was: the allocator's neighbours of every output keep a pattern."""
  import ctypes
  from tapnet_amd import _ffi
  lib, ctx = _ffi.load_library(), ctypes.c_void_p()
  cfg = _ffi.TapirCfg(1, 4, 12, 0, 20.0, 256, 256, _ffi.TAPIR_BF16)
  assert lib.tapir_create(ctypes.byref(ctx), ctypes.byref(cfg), 0) == 0
  gen = generator(2)
  (q, k, v), dout = attention_inputs(gen, torch.bfloat16, 2, 33, 77, 4, 2, 40, packed=False)
  guard = 1024

  def framed(shape, dtype):
    n = math.prod(shape)
    whole = torch.full((guard + n + guard,), 1234.0, dtype=dtype, device='cuda')
    whole[guard:guard + n] = math.nan
    return whole, whole[guard:guard + n].view(shape)
  a = _ffi.TapirAttnArgs(2, 33, 77, 4, 2, 40, 0.2)
  for name, t in (('q', q), ('k', k), ('v', v), ('dout', dout)):
    setattr(a, name, t.data_ptr())
    getattr(a, name + '_stride')[:] = t.stride()[:3]
  frames = {n: framed(t.shape, t.dtype) for n, t in (('out', q), ('dq', q), ('dk', k), ('dv', v))}
  frames['out_f32'], frames['stats'] = framed(q.shape, torch.float32), framed((2, 2, 66, 2), torch.float32)
  for n, (_, t) in frames.items():
    setattr(a, n, t.data_ptr())
  stream = torch.cuda.current_stream().cuda_stream
  for backward in (0, 1):
    nbytes = ctypes.c_uint64()
    assert lib.tapir_cross_attention_workspace(ctx, ctypes.byref(a), backward, ctypes.byref(nbytes)) == 0
    whole, work = framed((max(1, nbytes.value // 4),), torch.float32)
    a.workspace, a.workspace_bytes = work.data_ptr(), nbytes.value
    call = lib.tapir_cross_attention_backward if backward else lib.tapir_cross_attention
    assert call(ctx, ctypes.byref(a), stream) == 0
    torch.cuda.synchronize()
    assert (whole[:guard] == 1234).all() and (whole[-guard:] == 1234).all()
  for n, (whole, t) in frames.items():
    assert (whole[:guard] == 1234).all() and (whole[-guard:] == 1234).all(), n
    assert not torch.isnan(t.float()).any(), n
  lib.tapir_destroy(ctx)


def test_refusals(A):
  gen = generator(1)
  x = randn(gen, 2, 4, 2, 32)
  half = x.half()
  for call in (lambda: A.layer_norm(half), lambda: A.layer_norm(x.cpu()), lambda: A.layer_norm(x, torch.ones(31, device='cuda')),
               lambda: A.layer_norm(x, torch.ones(32, device='cuda').bfloat16()), lambda: A.layer_norm(x, eps=-1.0),
               lambda: A.layer_norm(x, torch.ones(32)), lambda: A.layer_norm(x[..., :0])):
    with pytest.raises(ValueError):
      call()
  with pytest.raises(TypeError):
    A.layer_norm([1.0])
  p = torch.zeros(4, 3, device='cuda')
  for call in (lambda: A.rotary_positions(half, p), lambda: A.rotary_positions(x[0], p), lambda: A.rotary_positions(x, p[:3]),
               lambda: A.rotary_positions(x, p.double()), lambda: A.rotary_positions(x, p.cpu()),
               lambda: A.rotary_positions(x, p.clone().requires_grad_()), lambda: A.rotary_positions(x, torch.zeros(4, 5, device='cuda')),
               lambda: A.rotary_positions(x, p, sections=[16, 8]), lambda: A.rotary_positions(x, p, sections=[16, 8, 10]),
               lambda: A.rotary_positions(x, p, sections=[11, 11, 10]), lambda: A.rotary_positions(x, p, base=0.0),
               lambda: A.rotary_positions(x, p, base=(1.0, 2.0)), lambda: A.rotary_positions(x, torch.zeros(3, 4, 3, device='cuda')),
               lambda: A.rotary_positions(randn(gen, 1, 4, 1, 258), p)):
    with pytest.raises(ValueError):
      call()
  lengths = torch.tensor([4, 4], dtype=torch.int32, device='cuda')
  for call in (lambda: A.cross_attention(half, half, half), lambda: A.cross_attention(x, x.bfloat16(), x.bfloat16()),
               lambda: A.cross_attention(x, x.cpu(), x.cpu()), lambda: A.cross_attention(x, x, x[:, :3]),
               lambda: A.cross_attention(x, x[:1], x[:1]), lambda: A.cross_attention(x[:, :, :1], x, x),
               lambda: A.cross_attention(x[..., :20], x[..., :20], x[..., :20]), lambda: A.cross_attention(x, x, x, scale=0.0),
               lambda: A.cross_attention(x, x, x, scale=math.nan), lambda: A.cross_attention(x, x, x, key_lengths=lengths.long()),
               lambda: A.cross_attention(x, x, x, key_lengths=lengths[:1]), lambda: A.cross_attention(x, x, x, key_lengths=lengths.cpu()),
               lambda: A.cross_attention(x, x, x, key_mask=torch.ones(2, 4, device='cuda')),
               lambda: A.cross_attention(x, x, x, key_mask=torch.ones(2, 5, dtype=torch.bool, device='cuda')),
               lambda: A.cross_attention(randn(gen, 1, 2, 1, 136), *[randn(gen, 1, 2, 1, 136)] * 2)):
    with pytest.raises(ValueError):
      call()
