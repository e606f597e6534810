"""Attention where its results are easily lost."""
import math

import numpy as np
import pytest
import torch

import ocnn
from attention_reference import visible
from test_gpu_attention import compare, inputs, run

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ---- values that are no numbers -------------------------------------------------------------------------------------
def row_by_row(q, k, v, see, grad):
  """The definition in 64 bits, every row from the keys that it sees alone: a row that sees nothing is zeros, and a visible
  value that is no number goes where its product goes (0 x inf is none either)."""
  scale = q.shape[2] ** -0.5
  q, k, v, grad, see = (t.detach().cpu() for t in (q, k, v, grad, see))
  q, k, v, grad = (t.double() for t in (q, k, v, grad))
  group = q.shape[1] // k.shape[1]
  res = {'out': torch.zeros_like(q), 'dq': torch.zeros_like(q), 'dk': torch.zeros_like(k), 'dv': torch.zeros_like(v)}
  for i in range(q.shape[0]):
    keys = see[i].nonzero()[:, 0]
    for h in range(q.shape[1] if keys.numel() else 0):
      kh, vh, go = k[keys, h // group], v[keys, h // group], grad[i, h]
      p = torch.softmax((kh * q[i, h]).sum(1) * scale, 0)
      out = (p[:, None] * vh).sum(0)
      ds = p * ((vh * go).sum(1) - (out * go).sum()) * scale
      res['out'][i, h] = out
      res['dq'][i, h] = (ds[:, None] * kh).sum(0)
      res['dk'][keys, h // group] += ds[:, None] * q[i, h]
      res['dv'][keys, h // group] += p[:, None] * go
  return res


def spoil(what, q, k, v, g):
  if what == 'query':
    q[40], q[90, 1] = math.nan, math.nan
  elif what == 'key':                         # (seen by 32 .. 48 both ways: by 48 as the first of its window)
    k[40] = math.nan
    k[100, :, 3] = math.inf
  elif what == 'all keys minus infinity':     # (30 .. 42 see nothing else)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    k[22:51, :, 0] = -math.inf
  elif what == 'value of a weak key':         # (its probability is 0 in 32 bits)
    q[:, :, 0], k[:, :, 0] = 30.0, 0.0
    k[60, :, 0], v[60, :, 5] = -60.0, math.inf
  elif what == 'gradient':
    g[70, 0], g[75, :, 2] = math.inf, math.nan
  else:
    g[:] = math.inf


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('dim', [32, 128])
@pytest.mark.parametrize('masked,causal', [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize('what', ['query', 'key', 'all keys minus infinity', 'value of a weak key', 'gradient', 'every gradient'])
def test_what_is_no_number_is_seen(dtype, dim, masked, causal, what):
  """Without first nodes, so that a row's first key may be the one that is no number.  What is finite in the definition is
  finite here, and what is not is not.  Off by a few roundings to the data's type, and by those of a score's terms in 32
  bits, which add up to less than 16 in size."""
  n, offsets = 130, [0, 70, 130]
  q, k, v, g = inputs(n, 2, 1, dim, dtype, 21)
  spoil(what, q, k, v, g)
  mask = None
  if masked:
    mask = torch.rand(n, generator=torch.Generator(device='cuda').manual_seed(3), device='cuda') < 0.6
    mask[:12], mask[40], mask[22] = False, True, True                       # (rows 0 .. 3 see nothing)
  got = run(q, k, v, offsets, g, window=9, causal=causal, mask=mask)
  quiet = run(q, k, v, offsets, window=9, causal=causal, mask=mask)['out']
  want = row_by_row(q, k, v, visible(n, offsets, 9, 0, causal, mask, 'cuda'), g)
  assert masked or not all(want[name].isfinite().all() for name in want)
  assert torch.equal(quiet.nan_to_num(), got['out'].nan_to_num())
  for name in want:
    value, fine = got[name].detach().double().cpu(), want[name].isfinite()
    assert torch.equal(value.isfinite(), fine), name
    if fine.any():
      off = (value - want[name])[fine].abs().max().item()
      assert off <= (16 * torch.finfo(dtype).eps + (dim + 4) * 2.0 ** -20) * want[name][fine].abs().max().item(), name


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_a_step_that_sees_minus_infinity_alone(dtype):
  """Scores of minus infinity and nothing else: softmax has no value there; a sequence that is passed over has zeros."""
  q, k, v, _ = inputs(3, 4, 2, 32, dtype)
  caches = [torch.randn(3, 40, 2, 32, device='cuda').to(dtype) for _ in range(2)]
  q[0, :, 0], k[0, :, 0], caches[0][0, :, :, 0] = 1.0, -math.inf, -math.inf
  lengths = torch.tensor([30, 30, -1], dtype=torch.int32, device='cuda')
  out = ocnn.octree_attention_step(q, k, v, *caches, lengths, 0)
  assert out[0].isnan().all() and out[1].isfinite().all() and not out[2].any()


@pytest.mark.parametrize('what', ['dO', 'k', 'v'])
def test_a_step_that_overflows_is_not_slow(what):
  """Values that are no numbers everywhere, as loss scaling brings them about, are no reason to form rows key by key (which took
  a hundred times as long): a pass takes no more than ten times one of numbers."""
  n = 20000
  q, k, v, g = inputs(n, 8, 2, 64, F16, 1)
  kw = dict(window=500, sinks=2)
  bad = {'dO': g, 'k': k, 'v': v}[what].clone()
  spoilt = [bad.fill_(math.inf) if name == what else x for name, x in (('q', q), ('k', k), ('v', v), ('dO', g))]
  times = []
  for t in ([q, k, v, g], spoilt):
    run(*t[:3], [0, n], t[3], **kw)
    ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    ends[0].record()
    for _ in range(3):
      run(*t[:3], [0, n], t[3], **kw)
    ends[1].record()
    torch.cuda.synchronize()
    times.append(ends[0].elapsed_time(ends[1]))
  assert times[1] <= 10 * times[0], times


# ---- blocks that one of two tiles passes over ---------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('heads', [1, 2, 4])
@pytest.mark.parametrize('masked', [None, 0.5])
def test_first_nodes_around_the_border_of_two_tiles(dtype, heads, masked):
  """Heads of 128: two tiles of 128 rows share their blocks of keys.  The sequence's first nodes lie on both sides of the shared
  windows' begin, two blocks that the second tile needs before it passes over some."""
  border = 256 // heads
  for start in range(border - 40, border, 3):
    for window in (1, 7, 30):
      compare([start, 2 * border], heads, 1, 128, dtype, window, 33, True, masked=masked, seed=start)
      compare([start, 2 * border], heads, 1, 104, dtype, window, 64, False, masked=masked, seed=start)


# ---- weak keys in float16 ---------------------------------------------------------------------------------------------
def weak_keys(n, dim, least):
  """One strong key of value 1 and n - 1 about 2^-25 as strong of value 16: keys, values, the output, and how far it may be off
  when probabilities are kept in float16 at a power of two where its smallest step is `least` of the strongest: half of that
  step each, u = 2^-11 of the larger ones and of the result, 2^-20 for the sums in 32 bits and (dim + 4) 2^-24 of a score."""
  gen = torch.Generator(device='cuda').manual_seed(1)
  k = torch.zeros(n, 1, dim, device='cuda', dtype=F16)
  k[1:, 0, 0] = -(16.5 + 2 * torch.rand(n - 1, generator=gen, device='cuda')).to(F16)
  v = torch.full_like(k, 16.0)
  v[0] = 1.0
  return (k, v) + weak_output(k, v, least)


def weak_output(k, v, least):
  """(output, bound) of weak_keys, for those keys and values."""
  p = torch.softmax(k[:, 0, 0].double(), 0)
  out = (p * v[:, 0, 0].double()).sum()
  heavy = out * (2.0 ** -11 + 2.0 ** -20 + (k.shape[2] + 4) * 2.0 ** -24 * 18.5)
  return out.item(), (2.0 ** -11 * out + heavy + 0.5 * least * v.double()[:, 0, 0].sum()).item()


@pytest.mark.parametrize('dim', [16, 64, 128])
def test_many_weak_keys_in_half(dim):
  """The reference may lie 2^8 below the maximum, never above it; p is kept at 2^7 p at least."""
  n = 100000
  k, v, value, bound = weak_keys(n, dim, 2.0 ** -24 / 2.0 ** 7)
  q = torch.zeros(n, 1, dim, device='cuda', dtype=F16)
  q[:, 0, 0] = 1.0
  out = ocnn.octree_attention(q, k, v, torch.tensor([0, n], dtype=torch.int32, device='cuda'), scale=1.0)
  assert value > 1.01 and (out.double() - value).abs().max().item() <= bound


@pytest.mark.parametrize('dim,n', [(8, 100000), (40, 40000), (72, 40000)])
def test_many_weak_keys_in_a_step_in_half(dim, n):
  """More sequences than there is room for clusters of several CTAs, so that four warps share a sequence: a strong key for
  each (rows come to them in sixteens), p at 2^15 p."""
  k, v, _, _ = weak_keys(n, dim, 0.0)
  k[0:64:16, 0, 0], v[0:64:16] = 0.0, 1.0
  value, bound = weak_output(k, v, 2.0 ** -24 / 2.0 ** 15)
  q = torch.zeros(600, 1, dim, device='cuda', dtype=F16)
  q[..., 0] = 1.0
  caches = [t[None].repeat(600, 1, 1, 1) for t in (k, v)]
  lengths = torch.full((600,), n - 1, dtype=torch.int32, device='cuda')
  new = [t[-1:].expand(600, 1, dim) for t in (k, v)]
  out = ocnn.octree_attention_step(q, *new, *caches, lengths, scale=1.0)
  assert (out.double() - value).abs().max().item() <= bound


# ---- many sequences, first nodes seen from far ------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('longest,count', [(40, 150), (24, 700), (17, 900)])
def test_first_nodes_of_many_short_sequences(dtype, longest, count):
  """Sequences shorter and longer than the window side by side, more of them than could be longer than it, and fewer."""
  lengths = np.random.default_rng(longest).integers(0, longest + 1, count)
  compare(list(lengths), 2, 1, 32, dtype, 16, 3, False)
  compare(list(lengths), 2, 1, 32, dtype, 1, 2, True, masked=0.8)


# ---- gradients that are not asked for ---------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_gradients_of_queries_alone(dtype):
  """Frozen keys and values: the same bits for the queries, and the keys' kernels do not run."""
  q, k, v, g = inputs(900, 4, 2, 32, dtype, 4)
  off = torch.tensor([0, 500, 900], dtype=torch.int32, device='cuda')
  kw = dict(window=40, sinks=2)
  want = run(q, k, v, [0, 500, 900], g, **kw)
  leaves = [t.detach().requires_grad_() for t in (q, k, v)]

  def launches(asked):
    given = [leaf if at in asked else leaf.detach() for at, leaf in enumerate(leaves)]
    out = ocnn.octree_attention(*given, off, **kw)
    before = ocnn.nn.launch_count()
    got = torch.autograd.grad(out, [given[at] for at in asked], g)
    for at, x in zip(asked, got):
      assert torch.equal(x, want[('dq', 'dk', 'dv')[at]])
    return ocnn.nn.launch_count() - before
  every = launches((0, 1, 2))
  assert launches((0,)) < every
  assert launches((1,)) == launches((2,)) == launches((1, 2)) == every


# ---- two streams at once ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_two_streams_at_once(dtype):
  """Forward passes and gradients of different inputs on two streams that do not wait for each other: the bits of the same
  passes one after the other."""
  kw = dict(window=300, sinks=4, causal=True)
  off = [0, 2500, 4100]
  sets = [inputs(4100, 4, 2, 64, dtype, seed) for seed in range(6)]
  want = [run(*s[:3], off, s[3], **kw) for s in sets]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in range(2)]
  got = []
  for at, s in enumerate(sets):
    with torch.cuda.stream(streams[at % 2]):
      got.append(run(*s[:3], off, s[3], **kw))
  torch.cuda.synchronize()
  for a, b in zip(got, want):
    for name in b:
      assert torch.equal(a[name], b[name]), name


# ---- the norm's gradients, as near as the kernel forms them -------------------------------------------------------------
def norm_gradients(x, r, w, eps, gy, gs):
  """{name: (value, bound)} in 64 bits.  The sum x + r enters as 32 bits hold it, so that a result is off by its own rounding
  and by those in 32 bits: up to 37 additions for a mean (32 in a thread, five between lanes; the root halves them) and a
  dozen products and sums, 2^-24 each: 2^-19 of every term; gw adds its rows besides."""
  u = torch.finfo(x.dtype).eps / 2
  x, r, gy, gs = (t.detach().double() for t in (x, r, gy, gs))
  wide = w.detach().double()
  x = x + r
  inv = (x.pow(2).mean(1, keepdim=True) + eps).rsqrt()
  unit, wg = x * inv, gy * wide
  g = gs + inv * (wg - unit * (wg * unit).mean(1, keepdim=True))
  heavy = gs.abs() + inv * (wg.abs() + unit.abs() * (wg * unit).abs().mean(1, keepdim=True))
  gw, terms = (gy * unit).sum(0), (gy * unit).abs().sum(0)
  return {'g': (g, u * g.abs() + 2.0 ** -19 * heavy),
          'gw': (gw, torch.finfo(w.dtype).eps / 2 * gw.abs() + (2.0 ** -19 + x.shape[0] * 2.0 ** -24) * terms)}


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('rows,channels', [(40, 8), (61, 96), (64, 128), (33, 1000)])
def test_norm_gradients_from_the_unrounded_sum(dtype, rows, channels):
  """A gradient formed from the stored sum, which is rounded to 16 bits, is outside of these bounds: shown beside."""
  make = lambda seed: torch.randn(rows, channels, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda')
  x, r, gy, gs = make(0).to(dtype), (3 * make(1)).to(dtype), make(2).to(dtype), make(3).to(dtype)
  w = (1 + 0.2 * make(4)[0]).contiguous()
  leaves = [t.detach().requires_grad_() for t in (x, r, w)]
  gx, gr, gw = torch.autograd.grad(ocnn.add_rms_norm(*leaves, 1e-5), leaves, (gy, gs))
  want = norm_gradients(x, r, w, 1e-5, gy, gs)
  least = torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
  for got, name in ((gx, 'g'), (gr, 'g'), (gw, 'gw')):
    off = (got.double() - want[name][0]).abs()
    assert bool((off <= want[name][1] + least).all()), (name, (off / want[name][1]).max().item())
  stored = norm_gradients((x + r), torch.zeros_like(r), w, 1e-5, gy, gs)['gw'][0]
  assert bool(((stored - want['gw'][0]).abs() > want['gw'][1]).any())
