"""Cross attention on the host emulator against tests/attention_tight.py: long sums, tokens that each show in a result, and what the
bounds reject (mistakes planted in the oracle)."""
import pytest
import torch

from tests import attention_tight as N
from tests import test_attention_emulated as E

DTYPES, IDS = E.DTYPES, E.IDS


def all_of(k):
  return torch.ones(k.shape[:2], dtype=torch.bool)


def compare(c, q, k, v, dout, keep=None, **how):
  got = E.run_attention(c, q, k, v, dout=dout, **how)
  want = N.attention(q, k, v, all_of(k) if keep is None else keep, q.shape[-1] ** -0.5, dout)
  for name, g, w in zip(('out', 'dq', 'dk', 'dv'), got, want[1:]):
    N.check(name, g, w)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('keys,heads,kv_heads,dim', [(65, 1, 1, 32), (700, 2, 1, 64), (2111, 1, 1, 40), (1025, 1, 1, 128), (640, 1, 1, 96)])
def test_every_token_counts(dtype, keys, heads, kv_heads, dim):
  gen = torch.Generator().manual_seed(keys)
  q, k, v, dout, at = N.dominated(gen, dtype, 'cpu', keys, heads, kv_heads, dim, most=40)
  with E.Ctx(dtype) as c:
    compare(c, q, k, v, dout)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('queries,keys,dim', [(1, 4099, 64), (3, 2000, 32), (130, 600, 24)])
def test_rows_that_attend_to_everything(dtype, queries, keys, dim):
  """Probabilities of like size: the results are small sums of many terms, in which every rounding of p shows."""
  gen = torch.Generator().manual_seed(keys + 1)
  q, k, v, dout = E.inputs(gen, dtype, 1, queries, keys, 2, 1, dim)
  q = (0.3 * torch.randn(q.shape, generator=gen)).to(dtype)
  with E.Ctx(dtype) as c:
    compare(c, q, k, v, dout)


@pytest.mark.parametrize('dtype', E.DTYPES, ids=E.IDS)
def test_the_bounds_reject_mistakes(dtype):
  """Oracles that leave out the last 8 of 4099 keys, count one key twice, or round p and ds once to bf16 are outside the bounds."""
  keys, dim = 4099, 64
  gen = torch.Generator().manual_seed(5)
  q = (0.3 * torch.randn(1, 4, 1, dim, generator=gen)).to(dtype)
  k, v = (torch.randn(1, keys, 1, dim, generator=gen).to(dtype) for _ in range(2))
  dout = torch.randn(1, 4, 1, dim, generator=gen).to(dtype)
  want = N.attention(q, k, v, all_of(k), dim ** -0.5, dout)
  short = all_of(k)
  short[:, -8:] = False

  def rejected(values):
    out = []
    for (value, bound), other in zip(want[1:], values):
      out.append(bool(((other.to(dtype).double() - value).abs() > bound).any()))
    return out
  assert all(rejected([w[0] for w in N.attention(q, k, v, short, dim ** -0.5, dout)[1:]]))
  assert not any(rejected([w[0] for w in want[1:]]))
  twice = torch.cat([torch.arange(keys), torch.tensor([keys - 1])])
  kk, vv = k[:, twice], v[:, twice]
  other = [w[0] for w in N.attention(q, kk, vv, all_of(kk), dim ** -0.5, dout)[1:]]
  other[2:] = [torch.cat([t[:, :keys - 1], t[:, keys - 1:].sum(1, keepdim=True)], 1) for t in other[2:]]
  assert any(rejected(other))
  if dtype == torch.bfloat16:
    once = lambda t: t.to(torch.bfloat16).double()
    Q, K, V, D = (t.double()[0, :, 0] for t in (q, k, v, dout))
    p = torch.softmax(Q @ K.T * dim ** -0.5, -1)
    ds = p * (D @ V.T - (D * (p @ V)).sum(-1, keepdim=True)) * dim ** -0.5
    shape = lambda t: t[None, :, None]
    assert all(rejected([shape(once(p) @ V), shape(once(ds) @ K), shape(once(ds).T @ Q), shape(once(p).T @ D)]))


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('queries,keys,heads,kv_heads', [(1, 1, 1, 1), (3, 1, 2, 1), (1, 5, 2, 2), (4, 70, 2, 1)])
def test_axes_of_one_element_have_no_stride(dtype, queries, keys, heads, kv_heads):
  """One clip, token or head sliced out of rows of an odd pitch: nothing steps over that axis."""
  gen = torch.Generator().manual_seed(queries + keys)

  def odd(tokens, heads):
    t = torch.randn(1, tokens, heads, 32, generator=gen).to(dtype)
    strides = [643, heads * 32 if tokens > 1 else 37, 32 if heads > 1 else 35, 1]
    return t.as_strided(t.shape, strides)
  q, k, v, dout = odd(queries, heads), odd(keys, kv_heads), odd(keys, kv_heads), odd(queries, heads)
  with E.Ctx(dtype) as c:
    compare(c, q, k, v, dout)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('keys', [3, 2000])
def test_rows_without_a_softmax(dtype, keys):
  """A row whose allowed scores are all -inf, or hold a NaN or +inf, has no softmax: it is NaN and so is every gradient that it enters,
  as of a sum over its terms.  Rows beside it, and rows whose other scores are -inf, keep their values; a clip whose mask leaves
  nothing gives zeros."""
  gen = torch.Generator().manual_seed(keys)
  batch, queries, dim = 5, 4, 32
  q, k, v, dout = E.inputs(gen, dtype, batch, queries, keys, 1, 1, dim)
  k, v = k.contiguous(), v.contiguous()
  big = 2.0 ** 80                                           # (its square is past float32's range)
  q[:4, :, :, 0] = k[:4, :, :, 0] = 0.0
  q[0, 1, 0, 0], k[0, :, 0, 0] = big, -big                  # all scores of one row -inf
  q[1, 2, 0, 0], k[1, 0, 0, 0] = big, -big                  # one score of one row -inf
  q[2, 0, 0, 0] = float('nan')
  q[3, 3, 0, 0], k[3, -1, 0, 0] = big, big                  # one score of one row +inf
  mask = torch.ones(batch, keys, dtype=torch.bool)
  mask[4] = False
  k[4] = float('nan')
  with E.Ctx(dtype) as c:
    out, dq, dk, dv = (t.float() for t in E.run_attention(c, q, k, v, None, mask, dout=dout))
  lost = torch.zeros(batch, queries, dtype=torch.bool)
  lost[0, 1] = lost[2, 0] = lost[3, 3] = True
  assert torch.isnan(out[lost]).all() and torch.isnan(dq[lost]).all()
  assert torch.isfinite(out[~lost]).all() and torch.isfinite(dq[1:][~lost[1:]]).all()
  for b in (0, 2, 3):                                       # every key of the clip is a term of the row
    assert torch.isnan(dk[b]).all() and torch.isnan(dv[b]).all()
  assert torch.isfinite(dk[1]).all() and torch.isfinite(dv[1]).all()
  assert all((t[4] == 0).all() for t in (out, dq, dk, dv))


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('power', [-60, -30, 60])
def test_scales_at_the_ends_of_the_range(dtype, power):
  """Scores of ordinary size whose scale is far from one: the gradients are those of any other scale."""
  gen = torch.Generator().manual_seed(3)
  q, k, v, dout = E.inputs(gen, dtype, 1, 9, 900, 2, 1, 32)
  scale = 2.0 ** power
  q = (q.float() * 2.0 ** (-power - 2)).to(dtype)
  with E.Ctx(dtype) as c:
    got = E.run_attention(c, q, k, v, scale=scale, dout=dout)
  want = N.attention(q, k, v, all_of(k), scale, dout)
  for name, g, w in zip(('out', 'dq', 'dk', 'dv'), got, want[1:]):
    N.check(name, g, w)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_scales_out_of_range_are_refused(dtype):
  q = torch.zeros(1, 2, 1, 8, dtype=dtype)
  with E.Ctx(dtype) as c:
    for scale in (1.2e-38, 2.0 ** -61, 2.0 ** 61, 3e38, 0.0, -1.0):
      a = E.attn_args(q, q, q, scale=scale)
      a.out = a.out_f32 = a.stats = a.dout = a.dq = q.data_ptr()
      for name in ('tapir_cross_attention', 'tapir_cross_attention_backward'):
        assert c.raw(name, E.ctypes.byref(a), None) == E._ffi.TAPIR_ERR_INVALID
        assert b'scale' in c.lib.tapir_last_error(c.ctx)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('power', [8, 12, 16, 20, 26, 32, 40, 60])
@pytest.mark.parametrize('keys', [70, 3000])
def test_huge_scores(dtype, power, keys):
  """Scores of 2^power that are exact in float32 (small whole numbers times powers of two) and far apart: each row's softmax is one
  token, or the mean of two whose scores are the same.  Nothing is rounded on the way, so that only the operands' own count."""
  gen = torch.Generator().manual_seed(power)
  q = torch.zeros(1, 6, 1, 16)
  k = torch.zeros(1, keys, 1, 16)
  q[0, :, 0, 0] = torch.tensor([1.0, -1.0, 2.0, -2.0, 3.0, 1.0])
  k[0, :, 0, 0] = torch.randint(-100, 100, (keys,), generator=gen).float()
  k[0, 17, 0, 0], k[0, keys - 1, 0, 0] = 120.0, 120.0
  k[0, 3, 0, 0] = -127.0
  k = k * 2.0 ** (power // 2)
  q = q * 2.0 ** (power - power // 2)
  v = torch.randint(-8, 9, (1, keys, 1, 16), generator=gen).float()
  dout = torch.randint(-4, 5, (1, 6, 1, 16), generator=gen).float()
  with E.Ctx(dtype) as c:
    out, dq, dk, dv = (t.double() for t in E.run_attention(c, *(t.to(dtype) for t in (q, k, v)), scale=1.0, dout=dout.to(dtype)))
  V, D = v[0, :, 0].double(), dout[0, :, 0].double()
  p = torch.zeros(6, keys, dtype=torch.float64)
  p[[0, 2, 4, 5], 17] = p[[0, 2, 4, 5], keys - 1] = 0.5
  p[[1, 3], 3] = 1.0
  ds = p * (D @ V.T - (D * (p @ V)).sum(-1, keepdim=True))
  K, Q = k[0, :, 0].double(), q[0, :, 0].double()
  # each result: its own rounding, and 2^-18 of the magnitudes in its sum (dp and D are sums of 16 products)
  size = p * ((D.abs() @ V.abs().T) + (D.abs() * (p @ V.abs())).sum(-1, keepdim=True))
  want = dict(out=(p @ V, p @ V.abs()), dq=(ds @ K, size @ K.abs()), dk=(ds.T @ Q, size.T @ Q.abs()), dv=(p.T @ D, p.T @ D.abs()))
  for (name, (value, terms)), got in zip(want.items(), (out, dq, dk, dv)):
    excess = (got[0, :, 0] - value).abs() - (N.rounded(value, 2.0 ** -18 * terms, dtype))
    assert float(excess.nan_to_num(nan=float('inf')).max()) <= 0, (name, float(excess.max()))


def test_rotary_sines_and_cosines():
  """(1, 0) turned by the position itself.  Half a step of t (2^-25 from a half on) reaches a sine or cosine of a quarter turn with at
  most 0.71 of itself: 0.36 u (u = 2^-24); the last operation's rounding 0.5 u; t^2's 0.25 u, the sum before it 0.15 u; the
  cosine's first dropped term 0.41 u: 1.7 u together."""
  gen = torch.Generator().manual_seed(8)
  positions = (torch.rand(60000, 1, generator=gen) * 2000 - 1000)
  x = torch.zeros(1, 60000, 1, 2)
  x[..., 0] = 1.0
  with E.Ctx(torch.float32) as c:
    y = E.run_rotary(c, x, positions, [2], [10000.0], True).double()[0, :, 0]
  angle = positions.double()[:, 0]
  worst = max(float((y[:, 0] - angle.cos()).abs().max()), float((y[:, 1] - angle.sin()).abs().max()))
  assert worst <= 1.7 * 2.0 ** -24, worst * 2 ** 24


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_layer_norm_channels_past_32_bits_are_refused(dtype):
  """Columns are counted in 32 bits, a stride of threads past the last one included: from 2^30 on nothing is launched."""
  p, nbytes = torch.zeros(64).data_ptr(), E.ctypes.c_uint64()
  with E.Ctx(dtype) as c:
    for channels in (2 ** 30 + 1, 2 ** 31 - 256, 2 ** 31 - 1):
      for rc in (c.raw('tapir_layer_norm_workspace', 0, channels, E.ctypes.byref(nbytes)),
                 c.raw('tapir_layer_norm', p, channels, None, None, p, None, None, 0, channels, 1e-5, None),
                 c.raw('tapir_layer_norm_backward', p, channels, p, channels, None, p, p, p, None, None, 0, channels, None, 0, None)):
        assert rc == E._ffi.TAPIR_ERR_UNSUPPORTED
    assert c.raw('tapir_layer_norm_workspace', 1, 2 ** 30, E.ctypes.byref(nbytes)) == 0


def test_rows_of_a_padded_batch_are_not_split_on_a_guess():
  """Shares of dk and dv cost their memory and a join for every key, the padding's too: a padded batch that has nearly a tile for every
  compute unit goes without (the workspace tells), as the whole batch does; one with few tiles keeps them."""
  def shares(batch, queries, keys, heads, kv_heads, dim, padded):
    a = E._ffi.TapirAttnArgs(batch, queries, keys, heads, kv_heads, dim, 0.1)
    a.key_lengths = 16 if padded else None          # (not read)
    out = []
    with E.Ctx(torch.bfloat16) as c:
      for dk in (None, 16):
        a.dq, a.dk, a.dv, n = 16, dk, dk, E.ctypes.c_uint64()
        c('tapir_cross_attention_workspace', E.ctypes.byref(a), 1, E.ctypes.byref(n))
        out.append(n.value)
    return (out[1] - out[0]) // (8 * batch * keys * kv_heads * dim)
  assert shares(3, 1000, 8200, 4, 2, 128, True) == 0
  assert shares(3, 1000, 8200, 4, 2, 128, False) == 0
  assert shares(1, 40000, 4096, 1, 1, 64, False) > 1
  assert shares(3, 40000, 4096, 1, 1, 64, True) > 1 and shares(3, 3000, 1000, 2, 2, 128, True) > 4
