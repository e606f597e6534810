"""What is timed of the operators of an attention layer over octree nodes, through the package's public calls.

Every case is a dict of plain values; `kind` says which operator it drives:

  rotary     `ocnn.octree_rotary`: channels of every head turned by the node's x, y, z (and back: the gradient)
  norm       `ocnn.add_rms_norm`: the residual's addition and the root-mean-square norm (and its gradient)
  attention  `ocnn.octree_attention`: window of a shape's nodes plus its first ones (and its gradients)
  step       `ocnn.octree_attention_step`: one new node per sequence against a cache

Node counts follow the package's benchmark configurations (32 shapes x 20k points: 250 k nodes at depth 5, 60 k at depth 4;
a scene of 200k points) and widths its networks' (64 to 256 channels per node, 96 in the U-Net's decoder); heads of 128
channels, 16-bit caches and windows of some thousand nodes are generic sizes.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False
ocnn = None

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
EPS = 1e-6


def _package():
  """The package, for the calls that `own` makes."""
  global ocnn
  if ocnn is None:
    sys.path.insert(0, os.path.join(os.getcwd(), 'o-cnn_b200'))
    import ocnn as package
    ocnn = package
  return ocnn


def listed():
  return [
      # one new node for each of eight shapes being generated: nothing but latency
      dict(name='rotary_bf16_step_8', kind='rotary', rows=8, heads=12, dim=64, x=10, y=11, z=11, interleaved=False,
           depth=6, dtype='bf16', grad=False),
      # queries and keys of a batch's depth-5 level, inference
      dict(name='rotary_bf16_32x20k_d5', kind='rotary', rows=250117, heads=16, dim=32, x=5, y=5, z=6,
           interleaved=False, depth=5, dtype='bf16', grad=False),
      # a training layer of the U-Net's width, 96 channels in four heads of 24
      dict(name='rotary_f32_train_61k', kind='rotary', rows=61003, heads=8, dim=24, x=4, y=4, z=4,
           interleaved=True, depth=9, dtype='f32', grad=True),
      # one new node per shape again
      dict(name='norm_f16_step_8', kind='norm', rows=8, channels=256, dtype='f16', grad=False),
      # a training layer on a batch's depth-5 level
      dict(name='norm_bf16_train_250k', kind='norm', rows=250117, channels=128, dtype='bf16', grad=True),
      # the same in fp32 at the U-Net's width
      dict(name='norm_f32_train_61k', kind='norm', rows=61003, channels=96, dtype='f32', grad=True),
      # inference on a batch's depth-5 level: windows of 255 nodes, four heads of 32 channels
      dict(name='attn_bf16_32x20k_d5', kind='attention', batch=32, nodes=250117, heads=4, kv_heads=4, dim=32,
           window=128, sinks=0, causal=False, masked=False, dtype='bf16', grad=False),
      # a training layer on the depth-4 level: all of a level's nodes, the empty ones no keys, the first node seen by all
      dict(name='attn_bf16_train_d4', kind='attention', batch=32, nodes=60211, heads=8, kv_heads=8, dim=32,
           window=256, sinks=1, causal=False, masked=True, dtype='bf16', grad=True),
      # training in fp32, small batch, heads of 24 channels
      dict(name='attn_f32_train_8x', kind='attention', batch=8, nodes=20011, heads=4, kv_heads=4, dim=24,
           window=64, sinks=0, causal=False, masked=False, dtype='f32', grad=True),
      # training of a generative network: nodes in order, four query heads to a key head, wide heads
      dict(name='attn_f16_causal_train', kind='attention', batch=3, nodes=65539, heads=16, kv_heads=4, dim=128,
           window=1024, sinks=4, causal=True, masked=False, dtype='f16', grad=True),
      # serving: one shape
      dict(name='step_bf16_1', kind='step', batch=1, heads=8, kv_heads=8, dim=32, capacity=1024, window=256, sinks=1,
           rolled=False, dtype='bf16'),
      # serving: 64 sequences on rolling caches
      dict(name='step_bf16_64', kind='step', batch=64, heads=16, kv_heads=4, dim=128, capacity=4160, window=4096,
           sinks=4, rolled=True, dtype='bf16'),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  kind = rng.choice(['rotary', 'norm', 'attention', 'attention', 'attention', 'step'])
  dtype = rng.choice(['f32', 'bf16', 'bf16', 'f16'])
  if kind == 'rotary':
    dim = rng.choice([16, 24, 32, 48, 64, 128])
    heads = rng.randint(2, 24)
    most = 5e8 / (heads * dim * BYTES[dtype])
    third = dim // 6
    return dict(kind=kind, rows=_log(rng, 1, min(250000, most)), heads=heads, dim=dim,
                x=third, y=third, z=rng.randint(0, dim // 2 - 2 * third), interleaved=rng.random() < 0.5,
                depth=rng.randint(3, 10), dtype=dtype, grad=rng.random() < 0.5)
  if kind == 'norm':
    channels = 8 * _log(rng, 1, 256)
    most = 2e8 / (channels * BYTES[dtype])
    return dict(kind=kind, rows=_log(rng, 1, min(400000, most)), channels=channels, dtype=dtype,
                grad=rng.random() < 0.6)
  if kind == 'attention':
    dim = rng.choice([16, 24, 32, 48, 64, 96, 128])
    group = rng.choice([1, 1, 2, 4])
    kv_heads = rng.randint(1, 4)
    window = _log(rng, 8, 1024)
    causal = rng.random() < 0.5
    pairs = (1.8e11 if dtype != 'f32' else 2e10) / (dim * kv_heads * group * window * (1 if causal else 2))
    nodes = _log(rng, 40, min(250000, 200000000 // (dim * kv_heads * group), max(100, pairs)))
    return dict(kind=kind, batch=_log(rng, 1, min(48, nodes)), nodes=nodes, heads=kv_heads * group, kv_heads=kv_heads,
                dim=dim, window=window, sinks=rng.choice([0, 1, 4, 16]), causal=causal, masked=rng.random() < 0.3,
                dtype=dtype, grad=rng.random() < 0.6)
  dim = rng.choice([16, 32, 64, 128])
  kv_heads = rng.randint(1, 8)
  window = _log(rng, 16, 4096)
  sinks = rng.choice([0, 1, 4])
  rolled = rng.random() < 0.5
  capacity = window + sinks + rng.randint(0, 70) if rolled else _log(rng, window + sinks, 8192 + sinks)
  most = 270000000 // (capacity * dim * kv_heads)
  return dict(kind=kind, batch=_log(rng, 1, max(1, min(64, most))), heads=kv_heads * rng.choice([1, 2, 4, 7]),
              kv_heads=kv_heads, dim=dim, capacity=capacity, window=window, sinks=sinks, rolled=rolled, dtype=dtype)


def _lengths(case):
  """Nodes of every shape of the batch: uneven, and the same for a case whatever the seed."""
  rng = random.Random(case['nodes'] * 131 + case['batch'])
  share = [rng.uniform(0.3, 1.7) for _ in range(case['batch'])]
  cuts, at = [], 0.0
  for x in share:
    at += x
    cuts.append(int(case['nodes'] * at / sum(share)))
  cuts[-1] = case['nodes']
  return [b - a for a, b in zip([0] + cuts[:-1], cuts)]


def _kept_keys(length, window, sinks, causal):
  """How many pairs of a query and a key are visible in a sequence."""
  i = np.arange(length, dtype=np.int64)
  last = i if causal else np.minimum(length - 1, i + window - 1)
  pairs = int((last - np.maximum(0, i - window + 1) + 1).sum())
  for j in range(min(sinks, length)):
    pairs += max(0, length - j - window) + (0 if causal else max(0, j - window + 1))
  return pairs


def _sections(case):
  """Pairs of channels that each axis turns."""
  return [case['x'], case['y'], case['z']]


def work(case):
  size = BYTES[case['dtype']]
  kind = case['kind']
  if kind == 'rotary':
    n = case['rows'] * case['heads'] * case['dim']
    passes = 2 if case['grad'] else 1
    return dict(bytes=passes * 2 * n * size + case['rows'] * 12, flops=passes * 3 * n)
  if kind == 'norm':
    n = case['rows'] * case['channels']
    return dict(bytes=(7 if case['grad'] else 4) * n * size, flops=(14 if case['grad'] else 5) * n)
  if kind == 'attention':
    pairs = sum(_kept_keys(n, case['window'], case['sinks'], case['causal']) for n in _lengths(case))
    if case['masked']:
      pairs = int(0.6 * pairs)
    width = 2 * case['heads'] + 2 * case['kv_heads']        # q, out; k, v
    if case['grad']:
      width *= 2                                            # out's gradient, dq; dk, dv
    return dict(bytes=case['nodes'] * width * case['dim'] * size,
                flops=(14 if case['grad'] else 4) * case['dim'] * case['heads'] * pairs)
  keys = sum(_step_keys(case, p) for p in _step_positions(case))
  wide = keys * case['kv_heads'] * case['dim']
  return dict(bytes=(2 * wide + 2 * case['batch'] * (case['heads'] + case['kv_heads']) * case['dim']) * size,
              flops=4 * keys * case['heads'] * case['dim'])


def _step_positions(case):
  """Where every sequence stands: near the cache's end, or beyond it where the cache rolls."""
  rng = random.Random(case['capacity'] * 17 + case['batch'])
  lo, hi = (case['capacity'], 3 * case['capacity']) if case['rolled'] else (case['capacity'] // 2, case['capacity'])
  return [rng.randrange(lo, hi) for _ in range(case['batch'])]


def _step_keys(case, p):
  first = max(0, p - case['window'] + 1)
  return p - first + 1 + min(case['sinks'], first)


# ---- inputs -------------------------------------------------------------------------------------------------
def prepare(case, seed):
  gen = torch.Generator(device='cuda').manual_seed(seed)
  dtype = DTYPES[case['dtype']]
  normal = lambda *shape: torch.randn(*shape, generator=gen, device='cuda').to(dtype)
  kind = case['kind']
  s = dict(case=case)
  if kind == 'rotary':
    rows, heads, dim = case['rows'], case['heads'], case['dim']
    # queries and keys lie beside the values in the layer's one product
    s['data'] = normal(rows, heads + heads // 2, dim)[:, :heads]
    s['positions'] = torch.randint(0, 2 ** case['depth'], (rows, 3), generator=gen, device='cuda', dtype=torch.int32)
    freqs = np.concatenate([100.0 ** (-np.arange(n, dtype=np.float64) / max(n, 1)) for n in _sections(case)])
    s['freqs'] = torch.from_numpy(freqs).cuda()
    if case['grad']:
      s['grad'] = normal(rows, heads, dim)
      s['data'].requires_grad_()
  elif kind == 'norm':
    rows, channels = case['rows'], case['channels']
    s['data'], s['residual'] = normal(rows, channels), 2 * normal(rows, channels)
    s['weight'] = 1 + 0.1 * torch.randn(channels, generator=gen, device='cuda')
    if case['grad']:
      s['grad_norm'], s['grad_sum'] = normal(rows, channels), normal(rows, channels)
      for name in ('data', 'residual', 'weight'):
        s[name].requires_grad_()
  elif kind == 'attention':
    lengths = _lengths(case)
    n, dim = case['nodes'], case['dim']
    s['lengths'] = lengths
    s['offsets'] = torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32).cuda()
    s['q'], s['k'] = normal(n, case['heads'], dim), normal(n, case['kv_heads'], dim)
    s['v'] = normal(n, case['kv_heads'], dim)
    s['mask'] = torch.rand(n, generator=gen, device='cuda') < 0.6 if case['masked'] else None
    if case['grad']:
      s['grad'] = normal(n, case['heads'], dim)
      for name in 'qkv':
        s[name].requires_grad_()
  else:
    b, cap, dim = case['batch'], case['capacity'], case['dim']
    s['q'] = normal(b, case['heads'], dim)
    s['k'], s['v'] = normal(b, case['kv_heads'], dim), normal(b, case['kv_heads'], dim)
    s['k_cache'], s['v_cache'] = normal(b, cap, case['kv_heads'], dim), normal(b, cap, case['kv_heads'], dim)
    s['lengths'] = torch.tensor(_step_positions(case), dtype=torch.int32).cuda()
  return s


# ---- one pass -----------------------------------------------------------------------------------------------
def run(s):
  return (_run_own if own else _run_plain)(s)


def _run_own(s):
  lib = _package()
  case = s['case']
  kind = case['kind']
  if kind == 'rotary':
    out = lib.octree_rotary(s['data'], s['positions'], s['freqs'], _sections(case), interleaved=case['interleaved'])
    if not case['grad']:
      return out
    return (out.detach(),) + torch.autograd.grad(out, s['data'], s['grad'])
  if kind == 'norm':
    norm, total = lib.add_rms_norm(s['data'], s['residual'], s['weight'], EPS)
    if not case['grad']:
      return norm, total
    return (norm.detach(), total.detach()) + torch.autograd.grad(
        (norm, total), (s['data'], s['residual'], s['weight']), (s['grad_norm'], s['grad_sum']))
  if kind == 'attention':
    out = lib.octree_attention(s['q'], s['k'], s['v'], s['offsets'], case['window'], sinks=case['sinks'],
                               causal=case['causal'], mask=s['mask'])
    if not case['grad']:
      return out
    return (out.detach(),) + torch.autograd.grad(out, (s['q'], s['k'], s['v']), s['grad'])
  out = lib.octree_attention_step(s['q'], s['k'], s['v'], s['k_cache'], s['v_cache'], s['lengths'], case['window'],
                                  sinks=case['sinks'])
  return out, s['k_cache'], s['v_cache']


def _run_plain(s):
  with torch.no_grad():
    return dict(rotary=_plain_rotary, norm=_plain_norm, attention=_plain_attention, step=_plain_step)[s['case']['kind']](s)


def _plain_rotary(s):
  case = s['case']
  dtype = s['data'].dtype
  pairs = sum(_sections(case))
  axis = [a for a, n in enumerate(_sections(case)) for _ in range(n)]
  angle = s['positions'][:, axis].double() * s['freqs']                 # far positions lose their angle in 32 bits
  cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
  half = case['dim'] // 2
  if case['interleaved']:
    first, second = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
  else:
    first, second = slice(0, pairs), slice(half, half + pairs)

  def turned(x, sign):
    x = x.float()
    y = x.clone()
    y[..., first] = x[..., first] * cos - x[..., second] * (sign * sin)
    y[..., second] = x[..., second] * cos + x[..., first] * (sign * sin)
    return y.to(dtype)

  out = turned(s['data'], 1)
  return (out, turned(s['grad'], -1)) if case['grad'] else out


def _plain_norm(s):
  dtype = s['data'].dtype
  weight = s['weight']
  total = s['data'].float() + s['residual'].float()
  inv = torch.rsqrt((total * total).mean(1, keepdim=True) + EPS)
  unit = total * inv
  out = (unit * weight).to(dtype), total.to(dtype)
  if not s['case']['grad']:
    return out
  gy = s['grad_norm'].float()
  gw = (gy * unit).sum(0)
  gy = gy * weight
  g = (s['grad_sum'].float() + inv * (gy - unit * (gy * unit).mean(1, keepdim=True))).to(dtype)
  return out + (g, g, gw)


def _plain_attention(s):
  """Blocks of up to 2048 queries against the keys that one of them sees."""
  case = s['case']
  q, k, v = s['q'], s['k'], s['v']
  dtype = q.dtype
  n, heads, dim = q.shape
  kv = k.shape[1]
  group = heads // kv
  window, sinks, causal, mask = case['window'], case['sinks'], case['causal'], s['mask']
  scale = dim ** -0.5
  grad = case['grad']
  out = torch.zeros(n, heads, dim, dtype=torch.float32, device=q.device)
  if grad:
    dq = torch.zeros_like(out)
    dk = torch.zeros(n, kv, dim, dtype=torch.float32, device=q.device)
    dv = torch.zeros_like(dk)
  # [kv head, node, ...]: one product per block of queries and all heads
  rows = lambda x, a, b: x[a:b].float().transpose(0, 1)
  start = 0
  for length in s['lengths']:
    end = start + length
    for a in range(start, end, 2048):
      b = min(end, a + 2048)
      lo, hi = max(start, a - window + 1), b if causal else min(end, b + window - 1)
      first = min(start + sinks, lo)                       # first nodes that lie before the window of them all
      # and those behind it, where keys are seen both ways
      late = (start, start) if causal else (hi, max(hi, min(start + sinks, end)))
      parts = [(start, first), (lo, hi), late]
      j = torch.cat([torch.arange(x, y, device=q.device) for x, y in parts])
      i = torch.arange(a, b, device=q.device)[:, None]
      if causal:
        seen = (j <= i) & ((i - j < window) | (j < start + sinks))
      else:
        seen = ((i - j).abs() < window) | (j < start + sinks)
      if mask is not None:
        seen = seen & mask[j]
      seen = seen.repeat_interleave(group, 0)              # the group's heads of a node one after the other
      qb = q[a:b].float().view(b - a, kv, group, dim).transpose(0, 1).reshape(kv, -1, dim)
      kb = torch.cat([rows(k, x, y) for x, y in parts], 1)
      vb = torch.cat([rows(v, x, y) for x, y in parts], 1)
      score = (torch.bmm(qb, kb.transpose(1, 2)) * scale).masked_fill_(~seen, -math.inf)
      top = score.amax(2, keepdim=True)
      top = torch.where(top == -math.inf, torch.zeros_like(top), top)
      p = torch.exp(score - top)
      total = p.sum(2, keepdim=True)
      p = p / torch.where(total == 0, torch.ones_like(total), total)
      ob = torch.bmm(p, vb)
      back = lambda x: x.view(kv, b - a, group, dim).transpose(0, 1).reshape(b - a, heads, dim)
      out[a:b] = back(ob)
      if not grad:
        continue
      gb = s['grad'][a:b].float().view(b - a, kv, group, dim).transpose(0, 1).reshape(kv, -1, dim)
      ds = p * (torch.bmm(gb, vb.transpose(1, 2)) - (gb * ob).sum(2, keepdim=True)) * scale
      dq[a:b] = back(torch.bmm(ds, kb))
      gk, gv = torch.bmm(ds.transpose(1, 2), qb).transpose(0, 1), torch.bmm(p.transpose(1, 2), gb).transpose(0, 1)
      at = 0
      for x, y in parts:
        dk[x:y] += gk[at:at + y - x]
        dv[x:y] += gv[at:at + y - x]
        at += y - x
    start = end
  if not grad:
    return out.to(dtype)
  return out.to(dtype), dq.to(dtype), dk.to(dtype), dv.to(dtype)


def _slot(p, capacity, sinks):
  """Where a cache holds position p: the first nodes for good, the others in turn."""
  return torch.where(p < capacity, p, sinks + (p - sinks) % max(capacity - sinks, 1))


def _plain_step(s):
  case = s['case']
  b, heads, dim = s['q'].shape
  kv, capacity, sinks, window = case['kv_heads'], case['capacity'], case['sinks'], case['window']
  at = s['lengths'].long()
  batch = torch.arange(b, device=at.device)
  s['k_cache'][batch, _slot(at, capacity, sinks)] = s['k']
  s['v_cache'][batch, _slot(at, capacity, sinks)] = s['v']
  first = (at - window + 1).clamp(min=0)[:, None]
  recent = first + torch.arange(window, device=at.device)
  early = torch.arange(sinks, device=at.device).expand(b, sinks)
  p = torch.cat([early, recent], 1)
  seen = torch.cat([early < first, recent <= at[:, None]], 1)
  slot = _slot(torch.where(seen, p, torch.zeros_like(p)), capacity, sinks)
  k = s['k_cache'][batch[:, None], slot].float()                        # [b, n, kv, dim]
  v = s['v_cache'][batch[:, None], slot].float()
  q = s['q'].float().view(b, kv, heads // kv, dim)
  score = torch.matmul(q, k.permute(0, 2, 3, 1)) * dim ** -0.5           # [b, kv, group, n]
  score = score.masked_fill(~seen[:, None, None], -math.inf)
  p = torch.exp(score - score.amax(3, keepdim=True))
  out = torch.matmul(p / p.sum(3, keepdim=True), v.transpose(1, 2))
  return out.reshape(b, heads, dim).to(s['q'].dtype), s['k_cache'], s['v_cache']


# ---- the definitions in 64 bits -------------------------------------------------------------------------------
def exact(case, seed):
  s = prepare(case, seed)
  with torch.no_grad():
    return dict(rotary=_exact_rotary, norm=_exact_norm, attention=_exact_attention, step=_exact_step)[case['kind']](case, s)


def _exact_rotary(case, s):
  """Every pair of channels as a complex number, times exp(i angle)."""
  pairs, dim = sum(_sections(case)), case['dim']
  which = torch.tensor([a for a, n in enumerate(_sections(case)) for _ in range(n)], device='cuda', dtype=torch.long)
  turn = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'),
                     s['positions'].double().index_select(1, which) * s['freqs'])[:, None]

  def turned(x, turn):
    x = x.detach().double()
    pair = x.unflatten(2, (dim // 2, 2)) if case['interleaved'] else x.unflatten(2, (2, dim // 2)).transpose(2, 3)
    pair = torch.view_as_complex(pair.contiguous())
    pair = torch.view_as_real(torch.cat([pair[..., :pairs] * turn, pair[..., pairs:]], 2))
    return (pair if case['interleaved'] else pair.transpose(2, 3)).reshape(x.shape)

  out = turned(s['data'], turn)
  return (out, turned(s['grad'], turn.conj())) if case['grad'] else out


def _exact_norm(case, s):
  x = (s['data'].detach().double() + s['residual'].detach().double())
  w = s['weight'].detach().double()
  c = x.shape[1]
  length = torch.sqrt(x.pow(2).sum(1) / c + EPS)[:, None]               # y = w x / length
  if not case['grad']:
    return w * x / length, x
  gy = s['grad_norm'].double()
  along = (gy * w * x).sum(1, keepdim=True) / c
  g = s['grad_sum'].double() + gy * w / length - x * along / length ** 3
  return w * x / length, x, g, g, (gy * x / length).sum(0)


def _exact_attention(case, s):
  """Sequence by sequence and head by head group, all keys at once: softmax as exp(score - log sum exp)."""
  lengths = s['lengths']
  dim, heads, kv = case['dim'], case['heads'], case['kv_heads']
  if sum(n * n for n in lengths) * heads * (dim + 40) * (3 if case['grad'] else 1) > 3e13:
    return None
  q, k, v = (s[x].detach().double().transpose(0, 1) for x in 'qkv')
  k, v = k.repeat_interleave(heads // kv, 0), v.repeat_interleave(heads // kv, 0)
  out = torch.zeros_like(q)
  grads = [torch.zeros_like(q) for _ in range(3)] if case['grad'] else None
  go = s['grad'].double().transpose(0, 1) if case['grad'] else None
  at = 0
  for n in lengths:
    own_rows = slice(at, at + n)
    pos = torch.arange(n, device='cuda')
    step = max(1, int(6e7 / max(1, n * heads)))
    for a in range(0, n, step):
      block = slice(at + a, at + min(n, a + step))
      i = pos[a:a + step, None]
      apart = i - pos
      if case['causal']:
        hidden = (apart < 0) | ((apart >= case['window']) & (pos >= case['sinks']))
      else:
        hidden = (apart.abs() >= case['window']) & (pos >= case['sinks'])
      if s['mask'] is not None:
        hidden = hidden | ~s['mask'][own_rows]
      x = torch.matmul(q[:, block], k[:, own_rows].transpose(1, 2)) / math.sqrt(dim)
      x.masked_fill_(hidden, -math.inf)
      p = (x - torch.logsumexp(x, 2, keepdim=True)).exp_()
      p.nan_to_num_(0.0)                                                # rows that see nothing
      o = torch.matmul(p, v[:, own_rows])
      out[:, block] = o
      if grads is None:
        continue
      g = go[:, block]
      grads[2][:, own_rows] += torch.matmul(p.transpose(1, 2), g)
      dp = torch.matmul(g, v[:, own_rows].transpose(1, 2))
      dx = p * (dp - (dp * p).sum(2, keepdim=True)) / math.sqrt(dim)
      grads[0][:, block] = torch.matmul(dx, k[:, own_rows])
      grads[1][:, own_rows] += torch.matmul(dx.transpose(1, 2), q[:, block])
    at += n
  out = out.transpose(0, 1).contiguous()
  if grads is None:
    return out
  shared = lambda x: x.unflatten(0, (kv, heads // kv)).sum(1).transpose(0, 1).contiguous()
  return out, grads[0].transpose(0, 1).contiguous(), shared(grads[1]), shared(grads[2])


def _exact_step(case, s):
  """Sequence by sequence: the cache is unrolled into the positions it holds."""
  capacity, sinks, group = case['capacity'], case['sinks'], case['heads'] // case['kv_heads']
  out = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda')
  caches = [s['k_cache'].clone(), s['v_cache'].clone()]
  for b, p in enumerate(s['lengths'].tolist()):
    place = lambda x: x if x < sinks else sinks + (x - sinks) % (capacity - sinks)
    caches[0][b, place(p)], caches[1][b, place(p)] = s['k'][b], s['v'][b]
    slots = [place(x) for x in range(max(0, p - capacity), p + 1) if p - x < case['window'] and x >= sinks]
    slots += [x for x in range(min(sinks, p + 1))]
    k, v = (x[b, slots].double().repeat_interleave(group, 1) for x in caches)
    score = (k * s['q'][b].double()).sum(2) / math.sqrt(case['dim'])
    out[b] = (torch.softmax(score, 0)[:, :, None] * v).sum(0)
  return out, caches[0].double(), caches[1].double()
