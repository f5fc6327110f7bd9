"""Layer normalisation, rotary positions and cross attention (csrc/layer_norm.hpp, rotary.hpp, attention.hpp) through the C ABI
on the host emulator, against 64-bit forms with counted roundings (tests/attention_ref.py); the entry points' refusals."""
import ctypes
import mmap
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tapnet_amd import _ffi
from tests import attention_ref as R
from tests.emu_engine import emu_lib

DTYPES = [torch.float32, torch.bfloat16]
IDS = ['f32', 'bf16']


class Ctx:
  """A weightless context of the emulator library; tensors are torch CPU tensors."""

  def __init__(self, dtype):
    self.lib = emu_lib()
    cfg = _ffi.TapirCfg(1, 4, 12, 0, 20.0, 256, 256, _ffi.TAPIR_BF16 if dtype == torch.bfloat16 else _ffi.TAPIR_F32)
    self.ctx = ctypes.c_void_p()
    assert self.lib.tapir_create(ctypes.byref(self.ctx), ctypes.byref(cfg), 0) == 0

  def __enter__(self):
    return self

  def __exit__(self, *_):
    self.lib.tapir_destroy(self.ctx)

  def raw(self, name, *args):
    return getattr(self.lib, name)(self.ctx, *args)

  def __call__(self, name, *args):
    _ffi.check(self.lib, self.ctx, self.raw(name, *args), name)


def ptr(t):
  return None if t is None else t.data_ptr()


def aligned_empty(shape, dtype, fill=float('nan')):
  """Uninitialised results start as NaN, so that an element nobody writes shows."""
  return torch.full(shape, fill, dtype=dtype)


def workspace(nbytes):
  return torch.full((max(1, nbytes // 4),), float('nan'), dtype=torch.float32)


# ------------------------------------------------------------------------------------------------------ layer norm
def run_layer_norm(c, x, weight, bias, eps, dy):
  rows, n = x.shape
  y, dx = aligned_empty((rows, n), x.dtype), aligned_empty((rows, n), x.dtype)
  mean, rstd = aligned_empty((rows,), torch.float32), aligned_empty((rows,), torch.float32)
  c('tapir_layer_norm', x.data_ptr(), x.stride(0), ptr(weight), ptr(bias), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
    rows, n, eps, None)
  dg = None if weight is None else aligned_empty((n,), torch.float32)
  db = None if bias is None else aligned_empty((n,), torch.float32)
  nbytes = ctypes.c_uint64()
  c('tapir_layer_norm_workspace', rows, n, ctypes.byref(nbytes))
  work = workspace(nbytes.value)
  c('tapir_layer_norm_backward', x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0), ptr(weight), mean.data_ptr(),
    rstd.data_ptr(), dx.data_ptr(), ptr(dg), ptr(db), rows, n, work.data_ptr(), nbytes.value, None)
  return y, dx, dg, db


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('rows,channels,affine,pad', [
    (1, 1, 'full', 0), (3, 7, 'full', 0), (5, 8, 'none', 0), (9, 64, 'scale', 0), (33, 100, 'full', 4), (17, 256, 'full', 0),
    (6, 256, 'bias', 8), (5, 512, 'scale', 0), (4, 1001, 'full', 0), (3, 1024, 'full', 3), (2, 2048, 'full', 0),
    (3, 2056, 'full', 0), (2, 5001, 'full', 0), (0, 16, 'full', 0)])
def test_layer_norm(dtype, rows, channels, affine, pad):
  gen = torch.Generator().manual_seed(rows * 10007 + channels)
  randn = lambda *s: torch.randn(*s, generator=gen)
  x = (randn(rows, channels + pad) * 2 + randn(rows, 1) * 3).to(dtype)[:, :channels]
  dy = randn(rows, channels + pad).to(dtype)[:, :channels]
  weight = 1 + 0.3 * randn(channels) if affine in ('full', 'scale') else None
  bias = 0.3 * randn(channels) if affine in ('full', 'bias') else None
  with Ctx(dtype) as c:
    got = run_layer_norm(c, x, weight, bias, 1e-5, dy)
  want = R.layer_norm(x, weight, bias, 1e-5, dy)
  for name, g, w in zip(('y', 'dx', 'dweight', 'dbias'), got, want):
    assert (g is None) == (w is None)
    if g is not None:
      R.check(name, g, w)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_layer_norm_far_from_zero(dtype):
  """Rows whose mean is a thousand times their spread, and constant rows: the centred squares, not a difference of moments."""
  gen = torch.Generator().manual_seed(5)
  x = (1000 + torch.randn(8, 96, generator=gen)).to(dtype)
  x[3] = 7.0
  x[4] = 0.0
  dy = torch.randn(8, 96, generator=gen).to(dtype)
  weight = torch.rand(96, generator=gen)
  with Ctx(dtype) as c:
    got = run_layer_norm(c, x, weight, None, 1e-5, dy)
  for name, g, w in zip(('y', 'dx', 'dweight'), got, R.layer_norm(x, weight, None, 1e-5, dy)):
    R.check(name, g, w)
  assert torch.equal(got[0][3], torch.zeros(96, dtype=dtype))


# ------------------------------------------------------------------------------------------------ rotary positions
def run_rotary(c, x, positions, sections, bases, interleaved, inverse=False):
  batch, tokens, heads, dim = x.shape
  y = aligned_empty(x.shape, x.dtype)
  a = _ffi.TapirRotaryArgs(batch, tokens, heads, dim, len(sections), int(interleaved), int(inverse))
  a.section[:len(sections)], a.base[:len(sections)] = sections, bases
  a.x, a.x_stride[:], a.y = x.data_ptr(), x.stride()[:3], y.data_ptr()
  a.positions, a.positions_stride = positions.data_ptr(), positions.stride(0) if positions.ndim == 3 else 0
  c('tapir_rotary_positions', ctypes.byref(a), None)
  return y


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('interleaved', [False, True], ids=['halves', 'pairs'])
@pytest.mark.parametrize('batch,tokens,heads,dim,sections,shared', [
    (1, 1, 1, 2, [2], False), (2, 5, 3, 64, [22, 22, 20], True), (1, 9, 2, 64, [32, 16, 16], False), (2, 3, 2, 40, [20, 20], False),
    (1, 33, 1, 7, [2, 4], False), (1, 4, 8, 128, [16, 0, 48, 32], False), (1, 17, 2, 32, [32], False), (1, 2, 1, 256, [128, 128], False),
    (1, 0, 2, 32, [32], False)])
def test_rotary(dtype, interleaved, batch, tokens, heads, dim, sections, shared):
  gen = torch.Generator().manual_seed(dim * 31 + tokens)
  x = torch.randn(batch, tokens, heads, dim, generator=gen).to(dtype)
  shape = (tokens, len(sections)) if shared else (batch, tokens, len(sections))
  positions = torch.rand(shape, generator=gen) * 600 - 100
  bases = [10000.0, 100.0, 10000.0, 7.5][:len(sections)]
  with Ctx(dtype) as c:
    y = run_rotary(c, x, positions, sections, bases, interleaved)
    back = run_rotary(c, x, positions, sections, bases, interleaved, inverse=True)
  R.check('y', y, R.rotary(x, positions, sections, bases, interleaved))
  R.check('inverse', back, R.rotary(x, positions, sections, bases, interleaved, inverse=True))
  passed = sum(sections)
  assert torch.equal(y[..., passed:], x[..., passed:])


def test_rotary_far_positions_and_strides():
  """The hundred-thousandth frame (in 32 bits its angle would be off by 6e-3), negative positions, heads-first strides."""
  gen = torch.Generator().manual_seed(3)
  x = torch.randn(2, 3, 6, 48, generator=gen).transpose(1, 2)        # [2, 6, 3, 48]
  positions = torch.tensor([[0.0], [99999.0], [-99999.0], [1e6 + 0.5], [2.0 ** 24], [1e-30]]).expand(2, 6, 1).contiguous()
  with Ctx(torch.float32) as c:
    y = run_rotary(c, x, positions, [48], [10000.0], False)
  R.check('y', y, R.rotary(x, positions, [48], [10000.0], False))
  assert torch.equal(y[:, 0], x[:, 0])


# ------------------------------------------------------------------------------------------------- cross attention
def attn_args(q, k, v, lengths=None, mask=None, scale=None):
  a = _ffi.TapirAttnArgs(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3],
                         q.shape[3] ** -0.5 if scale is None else scale)
  a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
  a.q_stride[:], a.k_stride[:], a.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
  a.key_lengths, a.key_mask = ptr(lengths), ptr(mask)
  return a


def run_attention(c, q, k, v, lengths=None, mask=None, scale=None, dout=None, wanted='qkv'):
  a = attn_args(q, k, v, lengths, mask, scale)
  out = aligned_empty(q.shape, q.dtype)
  a.out = out.data_ptr()
  if dout is not None:
    out32, stats = aligned_empty(q.shape, torch.float32), aligned_empty((*q.shape[:3], 2), torch.float32)
    a.out_f32, a.stats = out32.data_ptr(), stats.data_ptr()
  nbytes = ctypes.c_uint64()
  c('tapir_cross_attention_workspace', ctypes.byref(a), 0, ctypes.byref(nbytes))
  work = workspace(nbytes.value)
  a.workspace, a.workspace_bytes = work.data_ptr(), nbytes.value
  c('tapir_cross_attention', ctypes.byref(a), None)
  if dout is None:
    return [out]
  a.dout, a.dout_stride[:] = dout.data_ptr(), dout.stride()[:3]
  grads = [aligned_empty(t.shape, t.dtype) for t in (q, k, v)]
  a.dq, a.dk, a.dv = (g.data_ptr() if n in wanted else None for n, g in zip('qkv', grads))
  c('tapir_cross_attention_workspace', ctypes.byref(a), 1, ctypes.byref(nbytes))
  work = workspace(nbytes.value)
  a.workspace, a.workspace_bytes = work.data_ptr(), nbytes.value
  c('tapir_cross_attention_backward', ctypes.byref(a), None)
  return [out, *grads]


def keep_mask(batch, keys, lengths, mask):
  keep = torch.ones(batch, keys, dtype=torch.bool) if mask is None else mask.clone()
  if lengths is not None:
    keep &= torch.arange(keys) < lengths[:, None].long()
  return keep


def inputs(gen, dtype, batch, queries, keys, heads, kv_heads, dim):
  randn = lambda *s: torch.randn(*s, generator=gen)
  q = randn(batch, queries, heads, dim)
  k, v = randn(batch, keys, 2, kv_heads, dim).to(dtype).unbind(2)     # as one projection leaves them: strided
  if keys:
    like = k[:, torch.randint(0, keys, (queries,), generator=gen)].float().repeat_interleave(heads // kv_heads, 2)
    q[:, ::2] = 0.5 * q[:, ::2] + like[:, ::2]
  return q.to(dtype), k, v, randn(batch, queries, heads, dim).to(dtype)


SHAPES = [  # batch, queries, keys, heads, kv_heads, dim
    (1, 1, 1, 1, 1, 32), (1, 3, 5, 2, 1, 8), (2, 33, 70, 4, 2, 40), (1, 130, 64, 1, 1, 64), (1, 7, 129, 6, 2, 128),
    (1, 64, 65, 2, 2, 96), (2, 1, 700, 4, 2, 64), (1, 40, 31, 3, 3, 16), (1, 35, 66, 2, 1, 72), (1, 3, 400, 2, 2, 88), (1, 5, 0, 2, 1, 32), (2, 0, 9, 2, 2, 32)]


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('batch,queries,keys,heads,kv_heads,dim', SHAPES)
def test_cross_attention(dtype, batch, queries, keys, heads, kv_heads, dim):
  gen = torch.Generator().manual_seed(queries * 1009 + keys)
  q, k, v, dout = inputs(gen, dtype, batch, queries, keys, heads, kv_heads, dim)
  with Ctx(dtype) as c:
    got = run_attention(c, q, k, v, dout=dout)
  want = R.attention(q, k, v, keep_mask(batch, keys, None, None), dim ** -0.5, dout)
  for name, g, w in zip(('out', 'dq', 'dk', 'dv'), got, want):
    R.check(name, g, w)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('how', ['lengths', 'mask', 'both'])
def test_cross_attention_masks(dtype, how):
  """Padding that holds NaN and infinities, clips without a token, lengths out of range, a mask that leaves nothing."""
  batch, queries, keys, heads, kv_heads, dim = 5, 9, 150, 4, 2, 24
  gen = torch.Generator().manual_seed(77)
  q, k, v, dout = inputs(gen, dtype, batch, queries, keys, heads, kv_heads, dim)
  lengths = torch.tensor([150, 71, 0, -4, 1000], dtype=torch.int32) if how != 'mask' else None
  mask = torch.rand(batch, keys, generator=gen) < 0.6 if how != 'lengths' else None
  if mask is not None:
    mask[1] = False
    mask[0, :64] = False
  keep = keep_mask(batch, keys, lengths, mask)
  bad = torch.tensor([float('nan'), float('inf'), -float('inf'), torch.finfo(dtype).max, torch.finfo(dtype).min])
  gone = (~keep).nonzero()
  k, v = k.clone(), v.clone()
  for t in (k, v):
    t[gone[:, 0], gone[:, 1]] = bad[torch.randint(0, 5, (len(gone), 1, 1), generator=gen)].to(dtype)
  with Ctx(dtype) as c:
    got = run_attention(c, q, k, v, lengths, mask, scale=0.3, dout=dout)
  want = R.attention(q, k, v, keep, 0.3, dout)
  for name, g, w in zip(('out', 'dq', 'dk', 'dv'), got, want):
    R.check(name, g, w)
  empty = ~keep.any(1)
  assert empty.any() and (got[0][empty] == 0).all() and (got[1][empty] == 0).all()
  assert (got[2][~keep] == 0).all() and (got[3][~keep] == 0).all()


@pytest.mark.parametrize('queries,keys', [(3, 300), (400, 200), (70, 1500)])
def test_cross_attention_many_clips(queries, keys):
  """More clips than a wave has lanes, of all lengths from none to whole: each is found, and what nobody sums is zero."""
  batch, heads, kv_heads, dim = 70 if keys < 1000 else 9, 1, 1, 8
  gen = torch.Generator().manual_seed(13)
  q, k, v, dout = inputs(gen, torch.bfloat16, batch, queries, keys, heads, kv_heads, dim)
  lengths = torch.randint(0, keys + 1, (batch,), generator=gen).to(torch.int32)
  lengths[0], lengths[1], lengths[-1], lengths[-2] = 0, keys, keys, 0
  with Ctx(torch.bfloat16) as c:
    got = run_attention(c, q, k, v, lengths, dout=dout)
  want = R.attention(q, k, v, keep_mask(batch, keys, lengths, None), dim ** -0.5, dout)
  for name, g, w in zip(('out', 'dq', 'dk', 'dv'), got, want):
    R.check(name, g, w)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('queries,keys', [(5, 90), (300, 40)])
def test_cross_attention_some_gradients(dtype, queries, keys):
  """dq alone and dk / dv alone give the bits of the whole backward pass."""
  gen = torch.Generator().manual_seed(14)
  q, k, v, dout = inputs(gen, dtype, 2, queries, keys, 4, 2, 24)
  lengths = torch.tensor([keys, 7], dtype=torch.int32)
  with Ctx(dtype) as c:
    whole = run_attention(c, q, k, v, lengths, dout=dout)
    for wanted in ('q', 'kv'):
      part = run_attention(c, q, k, v, lengths, dout=dout, wanted=wanted)
      for n, (g, w) in enumerate(zip(part[1:], whole[1:])):
        if 'qkv'[n] in wanted:
          assert torch.equal(g, w)
        else:
          assert torch.isnan(g.float()).all()    # not written


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_cross_attention_gradient_that_is_not_finite(dtype):
  """An infinite or NaN gradient of one query spoils what it enters, never the gradients of masked tokens (zeros)."""
  gen = torch.Generator().manual_seed(15)
  q, k, v, dout = inputs(gen, dtype, 1, 40, 100, 2, 1, 32)
  dout[0, 3, 0] = float('inf')
  dout[0, 4, 1, 5] = float('nan')
  mask = torch.rand(1, 100, generator=gen) < 0.5
  with Ctx(dtype) as c:
    out, dq, dk, dv = run_attention(c, q, k, v, None, mask, dout=dout)
  assert (dk[~mask] == 0).all() and (dv[~mask] == 0).all() and torch.isfinite(out.float()).all()
  fine = torch.ones(40, 2, dtype=torch.bool)
  fine[3, 0] = fine[4, 1] = False
  assert torch.isfinite(dq[0][fine].float()).all() and not torch.isfinite(dq[0][~fine].float()).all()


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_cross_attention_large_scores(dtype):
  """Scores in the hundreds, the largest key last: the running maximum moves in every tile."""
  gen = torch.Generator().manual_seed(9)
  keys = 300
  q = torch.randn(1, 6, 1, 32, generator=gen).abs().to(dtype)
  k = (torch.linspace(-8, 8, keys)[None, :, None, None] * torch.ones(1, keys, 1, 32)).to(dtype)
  v = torch.randn(1, keys, 1, 32, generator=gen).to(dtype)
  dout = torch.randn(1, 6, 1, 32, generator=gen).to(dtype)
  with Ctx(dtype) as c:
    got = run_attention(c, q, k, v, scale=2.0, dout=dout)
  for name, g, w in zip(('out', 'dq', 'dk', 'dv'), got, R.attention(q, k, v, torch.ones(1, keys, dtype=torch.bool), 2.0, dout)):
    R.check(name, g, w)


# ------------------------------------------------------------------------------------------------ reads stay inside
def before_a_guard_page(t):
  """A copy of the tensor whose last byte is followed by a page that may not be touched."""
  nbytes = t.numel() * t.element_size()
  pages = -(-nbytes // mmap.PAGESIZE)
  region = mmap.mmap(-1, (pages + 1) * mmap.PAGESIZE)
  start = ctypes.addressof(ctypes.c_char.from_buffer(region))
  libc = ctypes.CDLL(None, use_errno=True)
  assert libc.mprotect(ctypes.c_void_p(start + pages * mmap.PAGESIZE), ctypes.c_size_t(mmap.PAGESIZE), 0) == 0
  at = np.frombuffer(region, dtype=np.uint8, count=nbytes, offset=pages * mmap.PAGESIZE - nbytes)
  out = torch.from_numpy(at).view(t.dtype).view(t.shape)
  out.copy_(t)
  return out


def reads_up_to_the_last_byte():
  gen = torch.Generator().manual_seed(17)
  for dtype in DTYPES:
    for queries, keys, dim in ((64, 64, 96), (128, 192, 96), (70, 130, 72), (3, 64, 128), (33, 70, 40), (64, 64, 64), (1, 1, 8), (130, 257, 104)):
      q, k, v, dout = (before_a_guard_page(t.contiguous()) for t in inputs(gen, dtype, 1, queries, keys, 2, 1, dim))
      mask = before_a_guard_page(torch.ones(1, keys, dtype=torch.bool))
      lengths = before_a_guard_page(torch.tensor([keys, ], dtype=torch.int32))
      print(dtype, queries, keys, dim, flush=True)
      with Ctx(dtype) as c:
        run_attention(c, q, k, v, dout=dout)
        run_attention(c, q, k, v, lengths, mask, dout=dout)
        x = before_a_guard_page(torch.randn(1, 5, 2, dim, generator=gen).to(dtype))
        run_rotary(c, x, before_a_guard_page(torch.rand(1, 5, 1, generator=gen)), [dim // 2 // 2 * 2], [100.0], False)
        rows = before_a_guard_page(torch.randn(9, dim + 1, generator=gen).to(dtype))
        run_layer_norm(c, rows, before_a_guard_page(torch.rand(dim + 1, generator=gen)), None, 1e-5, rows)
        rows = before_a_guard_page(torch.randn(9, dim, generator=gen).to(dtype))
        run_layer_norm(c, rows, before_a_guard_page(torch.rand(dim, generator=gen)), None, 1e-5, rows)


def test_reads_stay_inside():
  """Inputs that end where memory ends, in a process of its own (a read behind them ends it)."""
  root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
  emu_lib()
  done = subprocess.run([sys.executable, '-c', 'from tests import test_attention_emulated as t; t.reads_up_to_the_last_byte(); print("all")'],
                        cwd=root, capture_output=True, text=True, timeout=600)
  assert done.returncode == 0 and done.stdout.endswith('all\n'), (done.returncode, done.stdout[-300:], done.stderr[-600:])


# ----------------------------------------------------------------------------------------------------- refusals
def test_refusals():
  """Every refused call gives its code and a message; nothing is launched (the emulator would fault on the null pointers)."""
  INV, UNS = _ffi.TAPIR_ERR_INVALID, _ffi.TAPIR_ERR_UNSUPPORTED
  x = torch.zeros(64)
  p = x.data_ptr()
  with Ctx(torch.float32) as c:
    ln = lambda *a: c.raw('tapir_layer_norm', *a)
    assert ln(None, 8, None, None, p, None, None, 2, 8, 1e-5, None) == INV
    assert ln(p, 8, None, None, p, None, None, -1, 8, 1e-5, None) == INV
    assert ln(p, 8, None, None, p, None, None, 2, 0, 1e-5, None) == INV
    assert ln(p, 8, None, None, p, None, None, 2, 8, float('nan'), None) == INV
    assert ln(p, 8, None, None, p, p, None, 2, 8, 1e-5, None) == INV
    assert b'mean and rstd' in c.lib.tapir_last_error(c.ctx)
    assert c.raw('tapir_layer_norm_backward', p, 8, p, 8, None, p, p, p, p, None, 2, 8, None, 0, None) == INV
    assert c.raw('tapir_layer_norm_backward', p, 8, p, 8, None, p, p, p, p, None, 2, 8, p, 4, None) == INV
    assert b'workspace' in c.lib.tapir_last_error(c.ctx)
    assert c.raw('tapir_layer_norm_workspace', 2, 8, None) == INV

    def rotary(**changes):
      a = _ffi.TapirRotaryArgs(1, 2, 1, 8, 1, 0, 0)
      a.section[0], a.base[0] = 8, 10000.0
      a.x = a.y = a.positions = p
      a.x_stride[:] = [16, 8, 8]
      for n, v in changes.items():
        if n in ('section', 'base'):
          getattr(a, n)[0] = v
        else:
          setattr(a, n, v)
      return c.raw('tapir_rotary_positions', ctypes.byref(a), None)
    assert rotary(section=7) == INV and rotary(section=10) == INV and rotary(section=-2) == INV
    assert rotary(base=0.0) == INV and rotary(base=float('inf')) == INV
    assert rotary(axes=0) == INV and rotary(axes=5) == INV and rotary(dim=258) == UNS and rotary(x=None) == INV
    assert rotary(batch=-1) == INV and c.raw('tapir_rotary_positions', None, None) == INV
    assert rotary(batch=1 << 41) == UNS and rotary(tokens=1 << 40, batch=1 << 20) == UNS

    def attend(backward=False, **changes):
      a = _ffi.TapirAttnArgs(1, 2, 2, 2, 1, 8, 1.0)
      for n in ('q', 'k', 'v', 'out', 'out_f32', 'stats', 'dout', 'dq', 'dk', 'dv', 'workspace'):
        setattr(a, n, p)
      a.workspace_bytes = 256
      for n in ('q', 'k', 'v', 'dout'):
        getattr(a, n + '_stride')[:] = [16, 8, 8]
      for n, v in changes.items():
        if n.endswith('_stride'):
          getattr(a, n)[1] = v
        else:
          setattr(a, n, v)
      return c.raw('tapir_cross_attention_backward' if backward else 'tapir_cross_attention', ctypes.byref(a), None)
    for back in (False, True):
      for dim in (0, 4, 12, 136):
        assert attend(back, dim=dim) == UNS
      for bad in (dict(kv_heads=0), dict(heads=3, kv_heads=2), dict(batch=-1), dict(queries=-1), dict(keys=-1), dict(scale=0.0),
                  dict(scale=-1.0), dict(scale=float('nan')), dict(q=None), dict(k=p + 4), dict(v=None), dict(q_stride=10),
                  dict(k_stride=9), dict(v_stride=7)):
        assert attend(back, **bad) == INV, bad
      assert attend(back, q_stride=1 << 22) == UNS and attend(back, k_stride=1 << 22) == UNS and attend(back, v_stride=-8) == UNS
      assert attend(back, queries=1 << 31) == UNS and attend(back, keys=1 << 31) == UNS and attend(back, batch=1 << 22) == UNS
    assert attend(out=None) == INV and attend(stats=None) == INV and attend(out_f32=None) == INV
    assert attend(True, stats=None) == INV and attend(True, out_f32=None) == INV and attend(True, dk=None) == INV
    assert attend(True, dv=None) == INV and attend(True, dout=None) == INV and attend(True, dout_stride=3) == INV
    assert attend(True, workspace=None) == INV and attend(True, workspace_bytes=4) == INV
    assert c.raw('tapir_cross_attention', None, None) == INV
    many = dict(keys=1 << 20, workspace=None)
    assert attend(**many) == INV and b'workspace' in c.lib.tapir_last_error(c.ctx)
  for name, args in (('tapir_layer_norm', (p, 8, None, None, p, None, None, 2, 8, 1e-5, None)),
                     ('tapir_rotary_positions', (None, None)), ('tapir_cross_attention', (None, None))):
    assert getattr(emu_lib(), name)(None, *args) == INV
