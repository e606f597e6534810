"""Attention over a window of nodes: against the definition in 64 bits, at the sizes and masks where it can go wrong."""
import itertools
import math

import numpy as np
import pytest
import torch

import ocnn
from attention_reference import attention, check, visible

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def offsets_of(lengths, first=0):
  return [first] + [first + int(x) for x in np.cumsum(lengths)]


def inputs(n, heads, kv, dim, dtype, seed=0, strided=False):
  gen = torch.Generator(device='cuda').manual_seed(seed)
  if strided:                      # slices of one product, as a layer has them
    x = torch.randn(n, heads + 2 * kv, dim, generator=gen, device='cuda').to(dtype)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
  else:
    q, k, v = (torch.randn(n, h, dim, generator=gen, device='cuda').to(dtype) for h in (heads, kv, kv))
  g = torch.randn(n, heads, dim, generator=gen, device='cuda').to(dtype)
  return q, k, v, g


def run(q, k, v, offsets, g=None, **kw):
  off = torch.tensor(offsets, dtype=torch.int32, device='cuda')
  if g is None:
    return {'out': ocnn.octree_attention(q, k, v, off, **kw)}
  leaves = [t.detach().requires_grad_() for t in (q, k, v)]
  out = ocnn.octree_attention(*leaves, off, **kw)
  dq, dk, dv = torch.autograd.grad(out, leaves, g)
  return {'out': out, 'dq': dq, 'dk': dk, 'dv': dv}


def compare(lengths, heads, kv, dim, dtype, window, sinks, causal, masked=None, first=0, tail=0, strided=False,
            scale=None, seed=0):
  offsets = offsets_of(lengths, first)
  n = offsets[-1] + tail
  q, k, v, g = inputs(n, heads, kv, dim, dtype, seed, strided)
  mask = None
  if masked is not None:
    mask = torch.rand(n, generator=torch.Generator(device='cuda').manual_seed(7), device='cuda') < masked
  got = run(q, k, v, offsets, g, window=window, sinks=sinks, causal=causal, mask=mask, scale=scale)
  want = attention(q, k, v, visible(n, offsets, window, sinks, causal, mask, 'cuda'), scale, g)
  for name in want:
    check(got[name], want[name], name)
  quiet = run(q, k, v, offsets, window=window, sinks=sinks, causal=causal, mask=mask, scale=scale)['out']
  assert torch.equal(quiet, got['out'])
  assert int(ocnn.tc_status(q.device).item()) == 0


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('dim', [16, 24, 32, 64, 96, 128])
def test_ragged_batch(dtype, causal, dim):
  """Sequences of no, one and many nodes, one that ends on a tile's border, nodes outside of every sequence."""
  compare([1, 0, 130, 126, 3, 300, 0, 0, 65, 1], 4, 4, dim, dtype, 50, 0, causal, first=5, tail=40, strided=True)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('window,sinks,causal', list(itertools.product([0, 1, 2, 64, 127, 700], [0, 1, 5, 64], [False, True])))
def test_windows_and_first_nodes(dtype, window, sinks, causal):
  compare([400, 70, 233], 2, 1, 32, dtype, window, sinks, causal)


@pytest.mark.parametrize('dtype', [F32, F16])
@pytest.mark.parametrize('heads,kv', [(1, 1), (2, 1), (3, 1), (6, 3), (7, 1), (8, 2), (12, 2), (16, 1)])
@pytest.mark.parametrize('causal', [False, True])
def test_shared_heads(dtype, heads, kv, causal):
  compare([190, 5, 77], heads, kv, 64, dtype, 33, 2, causal)


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('kept', [0.0, 0.03, 0.5, 1.0])
@pytest.mark.parametrize('window,sinks', [(1, 0), (9, 3), (0, 0)])
def test_masks_that_leave_rows_empty(dtype, kept, window, sinks):
  for causal in (False, True):
    compare([150, 1, 200], 2, 2, 32, dtype, window, sinks, causal, masked=kept)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('dim', [1, 7, 20, 30, 100, 127])
def test_odd_heads(dtype, dim):
  compare([90, 41], 3, 3, dim, dtype, 20, 1, False, strided=True)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('n', [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_lengths_around_a_tile(dtype, n):
  for causal in (False, True):
    compare([n], 2, 2, 32, dtype, 0, 0, causal)
    compare([n], 2, 2, 64, dtype, 100, 1, causal)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('dim', [32, 128])
def test_first_nodes_seen_from_far(dtype, causal, dim):
  """Sequences over several blocks of the far pass, several sequences in one, first nodes that the mask hides."""
  compare([1500, 30, 700, 512, 20, 1100], 4, 2, dim, dtype, 16, 4, causal, masked=0.8)
  compare([40, 300, 5, 1000], 2, 2, dim, dtype, 16, 7, causal)


@pytest.mark.parametrize('window,sinks', [(16, 4), (100, 64), (300, 1), (0, 0)])
@pytest.mark.parametrize('masked', [None, 0.6])
@pytest.mark.parametrize('heads,kv', [(2, 2), (8, 1)])
def test_wide_heads(window, sinks, masked, heads, kv):
  """Two tiles that share their copies of keys and values, of which each needs some."""
  for causal in (False, True):
    compare([700, 3, 400, 129], heads, kv, 128, BF16, window, sinks, causal, masked=masked)


def test_small_gradients_in_half():
  """float16 with gradients far below 1, over many keys: probabilities and their gradients are smaller than its smallest
  numbers, the results are not.  Where p and ds are rounded, the bounds count half a step of their own, not of float16's
  smallest number: they are kept at powers of two that bring them into its range (dq, dk: relative to the largest dO)."""
  n = 6000
  q, k, v, g = inputs(n, 1, 1, 64, F16, 11)
  q, v = 0.2 * q, 16 * v
  g = (g.float() * 2.0 ** -6).to(F16)
  got = run(q, k, v, [0, n], g)
  see = torch.ones(n, n, dtype=torch.bool, device='cuda')
  wide = {name: (value, bound) for name, (value, bound) in
          attention(q.float(), k.float(), v.float(), see, None, g.float()).items()}
  u = 2.0 ** -11
  for name, heavy in (('dv', 1.0), ('dq', 1.0), ('dk', 1.0)):
    value = wide[name][0]
    off = (got[name].double() - value).norm() / value.norm()
    step = 2.0 ** -25 * math.sqrt(value.numel()) / value.norm()           # (the result's own smallest numbers)
    assert off <= 3 * u + step, (name, off.item(), step.item())


def test_a_large_gradient_among_small_ones_in_half():
  """One node's gradient 2^16 times the others': what does not see it keeps its precision (as above)."""
  n = 3000
  q, k, v, g = inputs(n, 2, 1, 32, F16, 12)
  g = (g.float() * 2.0 ** -7).to(F16)
  g[1500] = 2.0 ** 9
  kw = dict(window=40, sinks=1, causal=False)
  got = run(q, k, v, [0, n], g, **kw)
  see = visible(n, [0, n], 40, 1, False, None, 'cuda')
  far = (torch.arange(n, device='cuda') - 1500).abs() > 600         # (its chunk of 256 nodes, and windows around it)
  far[0] = False                                                    # (the first node is seen by all)
  u = 2.0 ** -11
  for name, (value, _) in attention(q.float(), k.float(), v.float(), see, None, g.float()).items():
    rows = far if name in ('dk', 'dv') else torch.arange(n, device='cuda') != 1500
    off = (got[name].double() - value)[rows].norm() / value[rows].norm()
    step = 2.0 ** -25 * math.sqrt(value[rows].numel()) / value[rows].norm()
    assert off <= 3 * u + step, (name, off.item(), step.item())


def test_many_short_sequences():
  lengths = np.random.default_rng(3).integers(0, 4, 2500)
  for dtype in (F32, BF16):
    compare(list(lengths[:900]), 2, 1, 32, dtype, 2, 1, False)
    compare(list(lengths), 1, 1, 16, dtype, 0, 0, True)


def test_large_scores():
  """Scores far apart and far from zero: the running maximum, not the scores, decides what is kept."""
  q, k, v, g = inputs(300, 2, 2, 64, F32, 3)
  q, k = 6 * q, 6 * k
  off = [0, 300]
  got = run(q, k, v, off, g, window=120, causal=True)
  want = attention(q, k, v, visible(300, off, 120, 0, True, None, 'cuda'), None, g)
  for name in want:
    check(got[name], want[name], name)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_scale(dtype):
  compare([100, 99], 2, 2, 32, dtype, 40, 0, False, scale=0.01)
  compare([100, 99], 2, 2, 32, dtype, 40, 0, False, scale=-0.5)


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_hidden_values_have_no_say(dtype):
  """What lies behind the mask, outside of the window or in another sequence may be anything."""
  offsets, n = [0, 100, 180], 200
  q, k, v, g = inputs(n, 2, 2, 32, dtype, 5)
  mask = torch.ones(n, dtype=torch.bool, device='cuda')
  mask[10:14] = mask[150] = False
  kw = dict(window=8, sinks=1, causal=False, mask=mask)
  clean = run(q, k, v, offsets, g, **kw)
  k2, v2 = k.clone(), v.clone()
  k2[10:14], v2[10:14], k2[150], v2[150] = math.nan, math.inf, -math.inf, math.nan
  k2[180:], v2[180:] = math.nan, math.nan                # behind the last sequence
  got = run(q, k2, v2, offsets, g, **kw)
  for name in got:
    assert torch.equal(got[name], clean[name]), name
  v2, k2 = v.clone(), k.clone()
  v2[60], k2[61] = math.inf, math.nan                     # seen by the nodes 53 .. 68
  out = run(q, k2, v2, offsets, **kw)['out']
  far = torch.ones(n, dtype=torch.bool)
  far[53:69] = False
  rel = (out[far].float() - clean['out'][far].float()).abs().max().item()
  assert rel <= 4 * torch.finfo(dtype).eps * clean['out'].abs().max().item()
  assert not torch.isfinite(out[53:69].float()).all(2).any()


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('dim', [32, 128])
def test_hidden_values_have_no_say_in_gradients(dtype, dim):
  """A node whose values are not numbers spoils what it sees and what sees it, no other node and no other sequence."""
  offsets, n = [0, 150, 400], 400
  q, k, v, g = inputs(n, 4, 2, dim, dtype, 6)
  kw = dict(window=9, sinks=2, causal=False)
  clean = run(q, k, v, offsets, g, **kw)
  q2, v2 = q.clone(), v.clone()
  v2[60], q2[300] = math.inf, math.nan                   # 60 is seen by 52 .. 68, whose delta it spoils; 300 sees 292 .. 308
  got = run(q2, k, v2, offsets, g, **kw)
  rows = torch.arange(n)
  near = lambda at, w: (rows - at).abs() < w
  spoilt = {'out': near(60, 9) | (rows == 300), 'dq': near(60, 9) | (rows == 300),
            'dk': near(60, 17) | near(300, 9) | (rows < 2) | near(151, 2) & (rows >= 150),
            'dv': near(60, 17) | near(300, 9) | (rows < 2) | near(151, 2) & (rows >= 150)}
  for name in got:
    rest = ~spoilt[name]
    off = (got[name][rest].double() - clean[name][rest].double()).abs().max().item()
    assert off <= 16 * torch.finfo(dtype).eps * clean[name].abs().max().item(), name


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('layout', ['heads first', 'expanded keys', 'one head', 'wide rows'])
def test_layouts(dtype, layout):
  offsets, n = [0, 90, 201], 201
  q, k, v, g = inputs(n, 4, 2, 64, dtype, 1)
  if layout == 'heads first':
    q, k, v, g = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g))
  elif layout == 'expanded keys':
    k, g = k[:, :1].expand(n, 2, 64), g[:1].expand(n, 4, 64)
  elif layout == 'one head':
    q, k, v, g = q[:, :1], k[:, :1], v[:, 1:], g[:, 3:]
  else:
    q, k, v, g = (torch.cat([t, t, t], 2)[..., 64:128] for t in (q, k, v, g))
  kw = dict(window=40, sinks=1, causal=True)
  got = run(q, k, v, offsets, g, **kw)
  want = attention(q, k, v, visible(n, offsets, 40, 1, True, None, 'cuda'), None, g)
  for name in want:
    check(got[name], want[name], name)


def test_gradient_against_differences():
  """Directional derivatives: with steps of h the difference quotient is off by the third derivative's h^2 / 6 (about
  1e-4 of the value for scores of order one, h = 0.02) and by the sums' rounding over h (1e-6 / 0.02)."""
  q, k, v, g = inputs(150, 4, 2, 32, F32, 9)
  kw = dict(window=30, sinks=2, causal=True)
  off = [0, 70, 150]
  got = run(q, k, v, off, g, **kw)
  off = torch.tensor(off, dtype=torch.int32, device='cuda')
  f = lambda *t: (ocnn.octree_attention(*t, off, **kw).double() * g.double()).sum().item()
  for at, name in enumerate(('dq', 'dk', 'dv')):
    step = 0.02 * torch.randn_like((q, k, v)[at])
    up, down = [q, k, v], [q, k, v]
    up[at], down[at] = up[at] + step, down[at] - step
    slope = (got[name].double() * step.double()).sum().item()
    size = (got[name].norm() * step.norm()).item() / math.sqrt(step.numel())
    assert abs((f(*up) - f(*down)) / 2 - slope) <= 2e-2 * size


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_same_bits_every_time(dtype):
  q, k, v, g = inputs(1400, 4, 2, 32, dtype, 2)
  kw = dict(window=100, sinks=4, causal=True)
  a, b = (run(q, k, v, [0, 900, 1400], g, **kw) for _ in range(2))
  for name in a:
    assert torch.equal(a[name], b[name]), name


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_other_stream_and_graphs(dtype):
  """Two captured passes (forward and gradients) replayed in turn on new inputs, with eager calls on a side stream."""
  kw = dict(window=60, sinks=2, causal=False)
  off = [0, 210, 333]
  graphs = []
  for seed in (0, 1):
    q, k, v, g = inputs(333, 2, 2, 64, dtype, seed)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    offs = torch.tensor(off, dtype=torch.int32, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      ocnn.octree_attention(*leaves, offs, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      out = ocnn.octree_attention(*leaves, offs, **kw)
      grads = torch.autograd.grad(out, leaves, g)
    graphs.append((graph, leaves, g, out, grads, offs))
  for seed in (5, 6, 7):
    for graph, leaves, g, out, grads, _ in graphs:
      new = inputs(333, 2, 2, 64, dtype, seed)
      with torch.no_grad():
        for old, x in zip(leaves + [g], new):
          old.copy_(x)
      graph.replay()
    for graph, leaves, g, out, grads, _ in graphs:
      want = run(*[t.detach() for t in leaves], off, g, **kw)
      torch.cuda.synchronize()
      for x, name in zip((out,) + grads, ('out', 'dq', 'dk', 'dv')):
        assert torch.equal(x, want[name]), name


def test_empty_calls():
  for n in (0, 3):
    q, k, v, g = inputs(n, 2, 2, 32, BF16)
    got = run(q, k, v, [0], g)                             # no sequence at all
    assert all(not x.any() and x.shape[0] == n for x in got.values())


def test_refusals():
  q, k, v, _ = inputs(10, 4, 2, 32, BF16)
  off = torch.tensor([0, 10], dtype=torch.int32, device='cuda')
  ok = ocnn.octree_attention(q, k, v, off)
  assert ok.shape == q.shape
  bad = [(q.cpu(), k, v, off), (q, k.float(), v, off), (q, k[:9], v[:9], off), (q[:, :3], k, v, off), (q, k, v[..., :16], off),
         (q.double(), k.double(), v.double(), off), (q, k, v, off.long()), (q, k, v, off.cpu()), (q, k, v, off[:0]),
         (q[0], k, v, off)]
  for args in bad:
    with pytest.raises(RuntimeError):
      ocnn.octree_attention(*args)
  wide = torch.zeros(10, 1, 136, dtype=BF16, device='cuda')
  for kw in (dict(window=-1), dict(sinks=-1), dict(sinks=65), dict(mask=torch.ones(9, dtype=torch.bool, device='cuda')),
             dict(mask=torch.ones(10, device='cuda'))):
    with pytest.raises(RuntimeError):
      ocnn.octree_attention(q, k, v, off, **kw)
  with pytest.raises(RuntimeError):
    ocnn.octree_attention(wide, wide, wide, off)
  leaf = q.clone().requires_grad_()
  with pytest.raises(RuntimeError, match='differentiated again'):
    torch.autograd.grad(ocnn.octree_attention(leaf, k, v, off).sum(), leaf, create_graph=True)


# ---- one new node per sequence ------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('heads,kv,dim', [(2, 2, 16), (4, 1, 24), (7, 1, 32), (4, 2, 64), (12, 1, 96), (8, 2, 128)])
@pytest.mark.parametrize('window,sinks,capacity', [(0, 0, 64), (20, 0, 64), (20, 3, 23), (7, 2, 30), (64, 4, 40)])
def test_steps(dtype, heads, kv, dim, window, sinks, capacity):
  """Node by node, sequences at different places, against causal attention over the nodes so far."""
  batch, steps = 3, 40
  q, k, v, _ = inputs(batch * steps, heads, kv, dim, dtype, 4, strided=True)
  q, k, v = (t.view(batch, steps, -1, dim) if t.is_contiguous() else t.unflatten(0, (batch, steps)) for t in (q, k, v))
  caches = [torch.full((batch, capacity, kv, dim), math.nan, dtype=dtype, device='cuda') for _ in range(2)]
  lengths = torch.zeros(batch, dtype=torch.int32, device='cuda')
  lead = [0, 0, -5]                                        # the last one starts five steps late
  for t in range(steps):
    lengths.copy_(torch.tensor([t + x for x in lead]))
    at = [max(0, t + x) for x in lead]
    pick = lambda x: torch.stack([x[b, p] for b, p in enumerate(at)])
    out = ocnn.octree_attention_step(pick(q), pick(k), pick(v), *caches, lengths, window, sinks=sinks)
    if t % 3 and t < steps - 3:
      continue
    for b, p in enumerate(at):
      if t + lead[b] < 0:
        assert not out[b].any()
        continue
      see = visible(p + 1, [0, p + 1], window, sinks, True, None, 'cuda')
      want = attention(q[b, :p + 1], k[b, :p + 1], v[b, :p + 1], see)['out']
      check(out[b], (want[0][p], want[1][p]), 'step %d sequence %d' % (t, b))


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_step_long_cache(dtype):
  """Long caches, split over the CTAs of a cluster, and the newest node only."""
  for batch, window, n in ((1, 0, 5000), (2, 3000, 4000), (1, 1, 300), (40, 0, 700)):
    q, k, v, _ = inputs(batch * n, 4, 2, 64, dtype, 8)
    k, v, q = (t.view(batch, n, -1, 64) for t in (k, v, q))
    caches = [t.clone() for t in (k, v)]
    caches[0][:, n - 1], caches[1][:, n - 1] = math.nan, math.nan
    lengths = torch.full((batch,), n - 1, dtype=torch.int32, device='cuda')
    out = ocnn.octree_attention_step(q[:, -1], k[:, -1], v[:, -1], *caches, lengths, window)
    assert torch.equal(caches[0], k) and torch.equal(caches[1], v)
    for b in range(batch):
      see = torch.ones(1, n, dtype=torch.bool, device='cuda')
      if window:
        see[:, :n - window] = False
      pair = attention_row(q[b, -1:], k[b], v[b], see)
      check(out[b:b + 1], pair, 'sequence %d of %d' % (b, batch))


def attention_row(q, k, v, see):
  """attention() for one query against n keys."""
  n = k.shape[0]
  got = attention(q.expand(n, -1, -1), k, v, see.expand(n, n))['out']
  return got[0][:1], got[1][:1]


def test_step_full_cache_and_refusals():
  q, k, v, _ = inputs(2, 4, 2, 32, BF16)
  caches = [torch.randn(2, 8, 2, 32, device='cuda').to(BF16) for _ in range(2)]
  before = [c.clone() for c in caches]
  lengths = torch.tensor([8, 7], dtype=torch.int32, device='cuda')
  out = ocnn.octree_attention_step(q, k, v, *caches, lengths, 0)
  assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
  assert all(torch.equal(c[0], b[0]) for c, b in zip(caches, before))
  assert torch.equal(caches[0][1, 7], k[1]) and torch.equal(caches[0][1, :7], before[0][1, :7])
  bad = [(q, k, v, caches[0], caches[1], lengths.long()), (q, k, v, caches[0][:1], caches[1][:1], lengths),
         (q, k, v, caches[0].float(), caches[1].float(), lengths), (q[:, :3], k, v, caches[0], caches[1], lengths),
         (q, k, v, caches[0][:, :1].expand(2, 8, 2, 32), caches[1], lengths), (q, k, v, caches[0], caches[1], lengths.cpu()),
         (q.cpu(), k, v, caches[0], caches[1], lengths), (q, k, v, caches[0], caches[0], lengths)]
  for args in bad:
    with pytest.raises(RuntimeError):
      ocnn.octree_attention_step(*args)
  with pytest.raises(RuntimeError, match='no gradient'):
    ocnn.octree_attention_step(q.clone().requires_grad_(), k, v, *caches, lengths)
  odd = torch.zeros(2, 2, 20, dtype=BF16, device='cuda')
  with pytest.raises(RuntimeError, match='16 bytes'):
    ocnn.octree_attention_step(odd, odd, odd, *[torch.zeros(2, 8, 2, 20, dtype=BF16, device='cuda')] * 2, lengths)


def test_step_in_a_graph():
  q, k, v, _ = inputs(2, 4, 2, 64, BF16)
  caches = [torch.zeros(2, 32, 2, 64, dtype=BF16, device='cuda') for _ in range(2)]
  twins = [c.clone() for c in caches]
  lengths = torch.zeros(2, dtype=torch.int32, device='cuda')
  graph = torch.cuda.CUDAGraph()
  ocnn.octree_attention_step(q, k, v, *[c.clone() for c in caches], lengths, 16)
  with torch.cuda.graph(graph):
    out = ocnn.octree_attention_step(q, k, v, *caches, lengths, 16)
    lengths += 1
  for t in range(40):
    for old, new in zip((q, k, v), inputs(2, 4, 2, 64, BF16, 100 + t)[:3]):
      old.copy_(new)
    graph.replay()
    want = ocnn.octree_attention_step(q, k, v, *twins, torch.full_like(lengths, t), 16)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(caches, twins))


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('dim,causal', [(32, True), (128, False), (20, True)])
def test_gradients_are_rounded_twice_at_most(dtype, dim, causal):
  """A gradient's terms are rounded once (p, ds), and so is their sum: two independent errors of one size, 1.42 times that of
  a result that is only rounded; no third of that size (out's own rounding, through delta) joins them: 1.74 with it."""
  lengths = [700, 300]
  offsets, n = offsets_of(lengths), 1000
  q, k, v, g = inputs(n, 4, 4, dim, dtype, 5)
  got = run(q, k, v, offsets, g, window=16, causal=causal)
  want = attention(q, k, v, visible(n, offsets, 16, 0, causal, None, 'cuda'), None, g)
  for name in ('out', 'dq', 'dk', 'dv'):
    value = want[name][0]
    once = (value.to(dtype).double() - value).norm()
    assert (got[name].detach().double() - value).norm() <= 1.5 * once, name
