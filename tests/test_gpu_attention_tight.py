"""Cross attention on an MI355X against tests/attention_tight.py: over many keys, with tokens at the ends of tiles and splits that each
show in a result."""
import pytest
import torch

from tests import attention_tight as N
from tests import test_gpu_attention as T

pytestmark = pytest.mark.gpu

DTYPES, IDS = T.DTYPES, T.IDS
A = T.A


def compare(A, q, k, v, dout, lengths=None, mask=None):
  inputs = [t.detach().requires_grad_() for t in (q, k, v)]
  keep = torch.ones(k.shape[:2], dtype=torch.bool, device='cuda') if mask is None else mask.clone()
  if lengths is not None:
    keep &= torch.arange(k.shape[1], device='cuda') < lengths[:, None].long()
  out = A.cross_attention(*inputs, key_lengths=lengths, key_mask=mask)
  grads = T.grads_of(out, inputs, dout)
  with torch.no_grad():
    want = N.attention(q, k, v, keep, q.shape[-1] ** -0.5, dout)
    for name, g, w in zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *grads), want[1:]):
      N.check(name, g, w)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('keys,heads,kv_heads,dim,most', [
    (4099, 2, 1, 64, 96), (20000, 4, 4, 64, 8), (20000, 2, 2, 32, 400), (49152, 1, 1, 64, 32), (8200, 4, 2, 128, 300), (3001, 2, 1, 96, 64),
    (129, 1, 1, 8, 64)])
def test_every_token_counts(A, dtype, keys, heads, kv_heads, dim, most):
  gen = T.generator(keys + dim)
  q, k, v, dout, _ = N.dominated(gen, dtype, 'cuda', keys, heads, kv_heads, dim, most)
  compare(A, q, k, v, dout)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_the_last_token_of_every_clip_counts(A, dtype):
  """A padded batch whose lengths end inside a tile, behind one and before one."""
  gen = T.generator(50)
  q, k, v, dout, _ = N.dominated(gen, dtype, 'cuda', 5000, 2, 1, 64, 8)
  lengths = torch.tensor([5000, 4097, 4096, 4095, 1, 65, 640, 2048], dtype=torch.int32, device='cuda')
  k, v = (t.expand(len(lengths), -1, -1, -1).contiguous() for t in (k, v))
  ends = k[torch.arange(len(lengths)), (lengths.long() - 1).tolist()][:, None].float().repeat_interleave(2, 2)
  q = (ends * (T.math.log(5000) + 2.2) * 8).to(dtype).expand(-1, 3, -1, -1).contiguous()
  compare(A, q, k, v, T.randn(gen, len(lengths), 3, 2, 64).to(dtype), lengths)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('queries,keys,heads,kv_heads,dim', [
    (1, 49152, 8, 2, 64), (3, 20000, 4, 4, 32), (256, 1024, 8, 8, 32), (1000, 4099, 2, 1, 64), (300, 3000, 2, 2, 128), (5, 4099, 2, 1, 104)])
def test_rows_that_attend_to_everything(A, dtype, queries, keys, heads, kv_heads, dim):
  """Probabilities of like size: the results are small sums of many terms, in which every rounding of p shows."""
  gen = T.generator(keys + queries)
  (_, k, v), dout = T.attention_inputs(gen, dtype, 1, queries, keys, heads, kv_heads, dim)
  compare(A, (0.3 * T.randn(gen, 1, queries, heads, dim)).to(dtype), k.detach(), v.detach(), dout)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_axes_of_one_element_have_no_stride(A, dtype):
  """One clip, token or head sliced out of rows of an odd pitch, for every tensor and for the result's gradient."""
  gen = T.generator(6)

  def one_token():
    t = T.randn(gen, 1, 1, 1, 35).to(dtype)[..., :32]
    assert t.stride() == (35, 35, 35, 1)
    return t

  def one_head(tokens):
    return T.randn(gen, 1, tokens, 3, 35).to(dtype)[:, :, :1, :32]

  def one_clip(tokens, heads):
    return T.randn(gen, 643 + tokens * heads * 32).to(dtype).as_strided((1, tokens, heads, 32), (643, heads * 32, 32, 1))
  for q, k, v, dout in ((one_token(), one_token(), one_token(), one_token()), (one_token(), one_head(5), one_clip(5, 1), one_token()),
                        (one_head(1), one_head(1), one_token(), one_head(1)), (one_clip(9, 4), one_clip(70, 2), one_clip(70, 2), one_clip(9, 4)),
                        (one_head(4), one_clip(3, 1), one_head(3), one_head(4)), (one_clip(1, 4), one_clip(33, 4), one_clip(33, 4), one_clip(1, 4))):
    compare(A, q, k, v, dout)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('keys', [3, 5000])
def test_rows_without_a_softmax(A, dtype, keys):
  """Rows whose allowed scores are all -inf, or hold a NaN or +inf: NaN, and every gradient that they enter; zeros where a mask
  leaves nothing, whatever the tokens hold."""
  gen = T.generator(keys)
  (q, k, v), dout = T.attention_inputs(gen, dtype, 5, 4, keys, 1, 1, 32, packed=False)
  big = 2.0 ** 80                                           # (its square is past float32's range)
  with torch.no_grad():
    q[:4, :, :, 0] = k[:4, :, :, 0] = 0.0
    q[0, 1, 0, 0], k[0, :, 0, 0] = big, -big                # all scores of one row -inf
    q[1, 2, 0, 0], k[1, 0, 0, 0] = big, -big                # one score of one row -inf
    q[2, 0, 0, 0] = T.math.nan
    q[3, 3, 0, 0], k[3, -1, 0, 0] = big, big                # one score of one row +inf
    k[4] = T.math.nan
  mask = torch.ones(5, keys, dtype=torch.bool, device='cuda')
  mask[4] = False
  y = A.cross_attention(q, k, v, key_mask=mask)
  dq, dk, dv = (t.float() for t in T.grads_of(y, [q, k, v], dout))
  out = y.detach().float()
  lost = torch.zeros(5, 4, dtype=torch.bool, device='cuda')
  lost[0, 1] = lost[2, 0] = lost[3, 3] = True
  assert torch.isnan(out[lost]).all() and torch.isnan(dq[lost]).all()
  assert torch.isfinite(out[~lost]).all() and torch.isfinite(dq[1:][~lost[1:]]).all()
  for b in (0, 2, 3):
    assert torch.isnan(dk[b]).all() and torch.isnan(dv[b]).all()
  assert torch.isfinite(dk[1]).all() and torch.isfinite(dv[1]).all()
  assert all((t[4] == 0).all() for t in (out, dq, dk, dv))


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('power', [8, 12, 16, 20, 26, 32, 60])
@pytest.mark.parametrize('keys,dim', [(70, 16), (3000, 64), (20000, 128), (900, 96)])
def test_huge_scores(A, dtype, power, keys, dim):
  """Scores of 2^power that are exact in float32 and far apart: each row's softmax is one token, or the mean of two whose scores
  are the same."""
  gen = T.generator(power)
  q, k = torch.zeros(1, 6, 1, dim, device='cuda'), torch.zeros(1, keys, 1, dim, device='cuda')
  q[0, :, 0, 0] = torch.tensor([1.0, -1.0, 2.0, -2.0, 3.0, 1.0])
  k[0, :, 0, 0] = torch.randint(-100, 100, (keys,), generator=gen, device='cuda').float()
  k[0, 17, 0, 0], k[0, keys - 1, 0, 0] = 120.0, 120.0
  k[0, 3, 0, 0] = -127.0
  q, k = q * 2.0 ** (power - power // 2), k * 2.0 ** (power // 2)
  v = torch.randint(-8, 9, (1, keys, 1, dim), generator=gen, device='cuda').float()
  dout = torch.randint(-4, 5, (1, 6, 1, dim), generator=gen, device='cuda').float()
  leaves = [t.to(dtype).requires_grad_() for t in (q, k, v)]
  y = A.cross_attention(*leaves, scale=1.0)
  got = [t.detach()[0, :, 0].double() for t in (y, *T.grads_of(y, leaves, dout.to(dtype)))]
  Q, K, V, D = (t[0, :, 0].double() for t in (q, k, v, dout))
  p = torch.zeros(6, keys, dtype=torch.float64, device='cuda')
  p[[0, 2, 4, 5], 17] = p[[0, 2, 4, 5], keys - 1] = 0.5
  p[[1, 3], 3] = 1.0
  ds = p * (D @ V.T - (D * (p @ V)).sum(-1, keepdim=True))
  # each result: its own rounding, and 2^-18 of the magnitudes in its sum (dp and D are sums of up to 128 exact products)
  size = p * ((D.abs() @ V.abs().T) + (D.abs() * (p @ V.abs())).sum(-1, keepdim=True))
  want = dict(out=(p @ V, p @ V.abs()), dq=(ds @ K, size @ K.abs()), dk=(ds.T @ Q, size.T @ Q.abs()), dv=(p.T @ D, p.T @ D.abs()))
  for (name, (value, terms)), g in zip(want.items(), got):
    excess = (g - value).abs() - N.rounded(value, 2.0 ** -18 * terms, dtype)
    assert float(excess.nan_to_num(nan=T.math.inf).max()) <= 0, (name, float(excess.max()))
