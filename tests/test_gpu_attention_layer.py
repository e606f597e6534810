"""Rotary positions, the residual's addition with the root-mean-square norm, and the layer they make with attention."""
import math

import pytest
import torch

import ocnn
from gpu_util import small_clouds

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def randn(*shape, dtype=F32, seed=0):
  return torch.randn(*shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda').to(dtype)


# ---- rotary positions -----------------------------------------------------------------------------------------------
def turned(x, positions, freqs, sections, interleaved, sign=1):
  """The definition in 64 bits."""
  axis = [a for a, n in enumerate(sections) for _ in range(n)]
  angle = sign * positions.double()[:, axis] * freqs
  cos, sin = angle.cos()[:, None], angle.sin()[:, None]
  t, half = len(axis), x.shape[2] // 2
  a, b = (slice(0, 2 * t, 2), slice(1, 2 * t, 2)) if interleaved else (slice(0, t), slice(half, half + t))
  x = x.detach().double()
  y = x.clone()
  y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
  return y


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dim,sections', [(2, [1]), (6, [1, 1, 1]), (16, [3, 2, 3]), (24, [4, 4, 4]), (32, [5, 5, 6]),
                                          (64, [0, 10, 3]), (100, [20, 0, 0, 30]), (128, [64]), (40, [0, 0])])
@pytest.mark.parametrize('n,heads', [(1, 1), (3, 7), (130, 4)])
def test_rotary(dtype, interleaved, dim, sections, n, heads):
  """Off by the rounding of the result (half a step, of float16's smallest number at least), and of a cosine or sine and
  two products in 32 bits."""
  u, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
  for floats in (False, True):
    wide = randn(n, heads + 2, dim, dtype=dtype, seed=n)
    x = wide[:, 1:heads + 1].detach().requires_grad_()
    pos = torch.randint(-100000, 100000, (n, len(sections)), device='cuda', dtype=torch.int32)
    if floats:
      pos = pos.float() / 64
    freqs = ocnn.rotary_freqs(sections, 1000.0)
    y = ocnn.octree_rotary(x, pos, freqs, sections, interleaved)
    g = randn(n, heads, dim, dtype=dtype, seed=1).transpose(0, 1).contiguous().transpose(0, 1)
    gx, = torch.autograd.grad(y, x, g)
    for got, src, sign in ((y, x, 1), (gx, g, -1)):
      want = turned(src, pos, freqs, sections, interleaved, sign)
      bound = u * want.abs() + 2.0 ** -21 * src.double().abs().amax(2, keepdim=True) + least
      assert bool(((got.detach().double() - want).abs() <= bound).all())


def test_rotary_passes_the_rest_through():
  x = randn(9, 2, 32, dtype=BF16)
  x[..., 4:16] = math.nan
  x[..., 20:] = math.inf
  pos = torch.zeros(9, 1, dtype=torch.int32, device='cuda')
  y = ocnn.octree_rotary(x, pos, ocnn.rotary_freqs([4]), [4])
  assert torch.equal(y.view(torch.int16), x.view(torch.int16))


def test_rotary_keeps_relative_positions():
  """q . k depends on the difference of the positions alone."""
  q, k = randn(1, 1, 48, seed=1), randn(1, 1, 48, seed=2)
  freqs = ocnn.rotary_freqs([8, 8, 8])
  a = torch.tensor([[3, 900, 41]], dtype=torch.int32, device='cuda')
  b = torch.tensor([[9, 870, 44]], dtype=torch.int32, device='cuda')
  dots = [(ocnn.octree_rotary(q, a + s, freqs, [8, 8, 8]) * ocnn.octree_rotary(k, b + s, freqs, [8, 8, 8])).sum().item()
          for s in (0, 1000, -1000000)]
  assert max(dots) - min(dots) <= 48 * 2.0 ** -21 * (q.norm() * k.norm()).item()


def test_rotary_refusals():
  x, pos = randn(5, 2, 16), torch.zeros(5, 2, dtype=torch.int32, device='cuda')
  freqs = ocnn.rotary_freqs([3, 3])
  assert ocnn.octree_rotary(x[:0], pos[:0], freqs, [3, 3]).shape == (0, 2, 16)
  for args in ((x.cpu(), pos, freqs, [3, 3]), (x[0], pos, freqs, [3, 3]), (x[..., :15], pos, freqs, [3, 3]),
               (x, pos[:4], freqs, [3, 3]), (x, pos, freqs, [6]), (x, pos, freqs.float(), [3, 3]), (x, pos, freqs, [3, 2]),
               (x, pos.long(), freqs, [3, 3]), (x, pos, ocnn.rotary_freqs([5, 5]), [5, 5]), (x, pos, freqs, [7, -1]),
               (x.double(), pos, freqs, [3, 3])):
    with pytest.raises(RuntimeError):
      ocnn.octree_rotary(*args)
  leaf = x.clone().requires_grad_()
  with pytest.raises(RuntimeError, match='differentiated again'):
    torch.autograd.grad(ocnn.octree_rotary(leaf, pos, freqs, [3, 3]).sum(), leaf, create_graph=True)


# ---- residual and norm ----------------------------------------------------------------------------------------------
def norm_reference(x, r, w, eps, gy=None, gs=None):
  """{name: (value, bound)}: u for each result's rounding; the sums of C squares in 32 bits are off by C 2^-24 at most
  (pairwise: far less), the gradient starts from the rounded sum: u of every term that holds it, twice in the statistics."""
  u = torch.finfo(x.dtype).eps / 2
  f32 = 2.0 ** -20
  x = x.detach().double() + (0 if r is None else r.detach().double())
  weight, w = w, w.detach().double()
  c = x.shape[-1]
  inv = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
  y = x * inv * w
  res = {'sum': (x, u * x.abs() + f32 * x.abs()), 'norm': (y, (u + f32) * y.abs())}
  if gy is None:
    return res
  gy, gs = gy.double(), gs.double()
  unit, wg = x * inv, gy * w
  g = gs + inv * (wg - unit * (wg * unit).mean(-1, keepdim=True))
  heavy = inv * (wg.abs() + unit.abs() * (wg * unit).abs().mean(-1, keepdim=True))
  res['g'] = g, u * g.abs() + 4 * (u + f32) * heavy + f32 * gs.abs()
  rows = x.reshape(-1, c).shape[0]
  gw, heavy = (gy * unit).reshape(-1, c).sum(0), (gy * unit).abs().reshape(-1, c).sum(0)
  res['gw'] = gw, torch.finfo(weight.dtype).eps / 2 * gw.abs() + (2 * u + 2 * f32 + rows * 2.0 ** -24) * heavy
  return res


def close(got, want, name):
  off = (got.detach().double() - want[0]).abs()
  least = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps / 2       # (half of the type's smallest number)
  assert bool((off <= want[1] + least + 1e-30).all()), '%s: %g over its bound' % (name, (off - want[1]).max().item())


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [1, 2, 37, 3001])
@pytest.mark.parametrize('channels', [1, 3, 8, 20, 64, 96, 100, 128, 256, 260, 1000, 2048, 5000, 9000])
def test_norm(dtype, rows, channels):
  if rows * channels > 4e6:
    rows = 300
  x, r = randn(rows, channels, dtype=dtype), 3 * randn(rows, channels, dtype=dtype, seed=1)
  gy, gs = randn(rows, channels, dtype=dtype, seed=2), randn(rows, channels, dtype=dtype, seed=3)
  for weight_dtype in {F32, dtype}:
    w = (1 + 0.2 * randn(channels, seed=4)).to(weight_dtype)
    leaves = [t.detach().requires_grad_() for t in (x, r, w)]
    y, s = ocnn.add_rms_norm(*leaves, 1e-5)
    gx, gr, gw = torch.autograd.grad((y, s), leaves, (gy, gs))
    want = norm_reference(x, r, w, 1e-5, gy, gs)
    for got, name in ((y, 'norm'), (s, 'sum'), (gx, 'g'), (gr, 'g'), (gw, 'gw')):
      close(got, want[name], name)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_norm_strides_and_parts(dtype):
  """Rows of a wider tensor, shifted by one value, three dimensions, no residual, one gradient only, zero rows."""
  wide, w = randn(50, 300, dtype=dtype), 1 + 0.2 * randn(64, seed=4)
  for x in (wide[:, :64], wide[:, 1:65], wide[::3, 8:72], wide[:, :64].reshape(5, 10, 64), wide[:1, :64].expand(50, 64)):
    leaf, weight = x.detach().requires_grad_(), w.detach().requires_grad_()
    y, s = ocnn.add_rms_norm(leaf, None, weight, 1e-6)
    assert s is leaf or s.data_ptr() == leaf.data_ptr()
    gy = randn(*x.shape, dtype=dtype, seed=5)
    want = norm_reference(x, None, w, 1e-6, gy, torch.zeros_like(gy))
    close(y, want['norm'], 'norm')
    gx, gw = torch.autograd.grad(y, (leaf, weight), gy)
    close(gx, want['g'], 'g')
    close(gw, want['gw'], 'gw')
  a, b = randn(7, 64, dtype=dtype).requires_grad_(), randn(7, 64, dtype=dtype, seed=1).requires_grad_()
  weight = w.detach().requires_grad_()
  y, s = ocnn.add_rms_norm(a, b, weight)
  ga, = torch.autograd.grad(s.sum(), a, retain_graph=True)
  assert torch.equal(ga, torch.ones_like(ga))
  gw, = torch.autograd.grad(y.sum(), weight)
  want = norm_reference(a, b, w, 1e-6, torch.ones_like(a), torch.zeros_like(a))
  close(gw, want['gw'], 'gw')
  empty = randn(0, 64, dtype=dtype).requires_grad_()
  y, s = ocnn.add_rms_norm(empty, empty.detach(), weight)
  gx, gw = torch.autograd.grad(y.sum(), (empty, weight))
  assert gx.shape == (0, 64) and not gw.any()
  zero = torch.zeros(4, 64, dtype=dtype, device='cuda')
  assert not ocnn.add_rms_norm(zero, zero, w)[0].any()


def test_norm_same_bits_and_graph():
  x, r, w = randn(5000, 128, dtype=BF16), randn(5000, 128, dtype=BF16, seed=1), randn(128, seed=2)
  leaves = [t.requires_grad_() for t in (x, r, w)]
  gy = randn(5000, 128, dtype=BF16, seed=3)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    y, s = ocnn.add_rms_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, gy)
  graph.replay()
  y2, s2 = ocnn.add_rms_norm(*leaves)
  again = torch.autograd.grad(y2, leaves, gy)
  for a, b in zip((y, s) + grads, (y2, s2) + again):
    assert torch.equal(a, b)


def test_norm_refusals():
  x, w = randn(5, 16, dtype=BF16), randn(16)
  for args in ((x.cpu(), None, w), (x, x[:4], w), (x, x.float(), w), (x, None, w[:15]), (x, None, w.half()),
               (x, None, w.cpu()), (x.double(), None, w), (x[:, :0], None, w[:0])):
    with pytest.raises(RuntimeError):
      ocnn.add_rms_norm(*args)
  leaf = x.clone().requires_grad_()
  with pytest.raises(RuntimeError, match='differentiated again'):
    torch.autograd.grad(ocnn.add_rms_norm(leaf, x, w)[0].sum(), leaf, create_graph=True)


# ---- the layer ------------------------------------------------------------------------------------------------------
def a_level(depth=5, nempty=False):
  clouds = [torch.from_numpy(ocnn_points(c)) for c in small_clouds(3, 3000)]
  octree = ocnn.points2octree_batch(clouds, depth, 2, False, False, False, False, 4, 0.1, 2.0, False, False, False)
  return octree, ocnn.octree_sequence(octree, depth, nempty)


def ocnn_points(cloud):
  from oracle import oracle as oc
  return oc.points_new(cloud[0], cloud[1])


@pytest.mark.parametrize('nempty', [False, True])
def test_sequence(nempty):
  octree, seq = a_level(5, nempty)
  index = ocnn.octree_property(octree, 'index', 5)
  xyz = ocnn.octree_decode_key(ocnn.octree_property(octree, 'xyz', 5))[:, :3].float()
  if nempty:
    kept = ocnn.octree_property(octree, 'child', 5) >= 0
    index, xyz = index[kept], xyz[kept]
  assert torch.equal(seq.positions, xyz) and seq.offsets.dtype == torch.int32
  counts = torch.bincount(index.long(), minlength=3)
  assert (seq.offsets[1:] - seq.offsets[:-1]).tolist() == counts.tolist() and int(seq.offsets[0]) == 0


def block_reference(block, data, seq, mask=None):
  """The block from torch operators in 64 bits."""
  at = block.attention
  p = {k: v.detach().double() for k, v in block.state_dict().items()}
  x = data.detach().double()[0, :, :, 0].t()
  norm = lambda x, w: x * (x.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * w
  qkv = norm(x, p['norm1.weight']) @ p['attention.qkv.conv1x1.weight'][:, :, 0].t()
  h, kv, dim = at.heads, at.kv_heads, at.dim
  rows = qkv.view(-1, h + 2 * kv, dim)
  q, k = (turned(t, seq.positions, at.freqs, at.sections, False) for t in (rows[:, :h], rows[:, h:h + kv]))
  from attention_reference import visible
  see = visible(x.shape[0], seq.offsets.tolist(), at.window, at.sinks, at.causal, mask, 'cuda')
  k, v = (t.transpose(0, 1).repeat_interleave(h // kv, 0) for t in (k, rows[:, h + kv:]))
  s = (q.transpose(0, 1) @ k.transpose(1, 2) / math.sqrt(dim)).masked_fill(~see, -math.inf)
  out = (torch.softmax(s, 2).nan_to_num(0.0) @ v).transpose(0, 1).reshape(x.shape[0], -1)
  x = x + out @ p['attention.proj.conv1x1.weight'][:, :, 0].t()
  mid = torch.relu(norm(x, p['norm2.weight']) @ p['fc1.conv1x1.weight'][:, :, 0].t() + p['fc1.conv1x1.bias'])
  return x + mid @ p['fc2.conv1x1.weight'][:, :, 0].t() + p['fc2.conv1x1.bias']


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_block(dtype):
  """All operators as a network has them, on an octree's level: forward in eval and training mode, and gradients that
  reach every parameter.  A value passes six roundings to the data's type on its way (norm, product, turn, attention,
  projection, sum), each of half a step of values a few times the result's size: 32 half steps of the largest."""
  torch.manual_seed(0)
  octree, seq = a_level(4)
  n = seq.positions.shape[0]
  block = ocnn.OctreeAttentionBlock(64, 4, kv_heads=2, window=40, sinks=1).cuda()
  data = randn(1, 64, n, 1, dtype=dtype).contiguous(memory_format=torch.channels_last)
  mask = ocnn.octree_property(octree, 'child', 4) >= 0
  want = block_reference(block, data, seq, mask)
  tol = 32 * max(torch.finfo(dtype).eps / 2, 2.0 ** -20) * want.abs().max().item()
  with torch.no_grad():
    quiet = block.eval()(data, seq, mask)
  assert (quiet[0, :, :, 0].t().double() - want).abs().max().item() <= tol
  leaf = data.clone().requires_grad_()
  out = block.train()(leaf, seq, mask)
  assert out.dtype == dtype and (out[0, :, :, 0].t().double() - want).abs().max().item() <= tol
  g = randn(*out.shape, dtype=dtype, seed=3)
  out.backward(g)
  assert leaf.grad is not None and all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())
  if dtype == F32:
    step = 0.01 * torch.randn_like(data)
    f = lambda x: (block(x, seq, mask).double() * g.double()).sum().item()
    with torch.no_grad():
      diff = (f(data + step) - f(data - step)) / 2
    slope = (leaf.grad.double() * step.double()).sum().item()
    assert abs(diff - slope) <= 2e-2 * (leaf.grad.norm() * step.norm()).item() / math.sqrt(step.numel()) + 1e-3 * abs(slope)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_node_by_node(dtype):
  """A causal network run on whole sequences and, from the middle on, node by node on rolling caches."""
  torch.manual_seed(1)
  lengths, extra = [50, 33, 7], 12
  blocks = [ocnn.OctreeAttentionBlock(32, 4, kv_heads=1, window=12, sinks=2, causal=True).cuda().eval() for _ in range(2)]
  total = [x + extra for x in lengths]
  pos = [torch.randint(0, 64, (x, 3), device='cuda').float() for x in total]
  data = [randn(x, 32, dtype=dtype, seed=i) for i, x in enumerate(total)]
  nodes = lambda rows: rows[None, :, None].permute(0, 3, 1, 2)
  offsets = lambda ls: torch.tensor([0] + [sum(ls[:i + 1]) for i in range(len(ls))], dtype=torch.int32, device='cuda')
  with torch.no_grad():
    x, seq = nodes(torch.cat(data)), ocnn.OctreeSequence(offsets(total), torch.cat(pos))
    for b in blocks:
      x = b(x, seq)
    whole = x[0, :, :, 0].t().split(total)
    caches = [ocnn.AttentionCache(3, 14, 1, 8, dtype) for _ in blocks]
    x = nodes(torch.cat([d[:n] for d, n in zip(data, lengths)]))
    seq = ocnn.OctreeSequence(offsets(lengths), torch.cat([p[:n] for p, n in zip(pos, lengths)]))
    for b, c in zip(blocks, caches):
      x = b(x, seq, cache=c)
    for t in range(extra):
      x = nodes(torch.stack([d[n + t] for d, n in zip(data, lengths)]))
      at = torch.stack([p[n + t] for p, n in zip(pos, lengths)])
      for b, c in zip(blocks, caches):
        x = b.step(x, at, c)
      got = x[0, :, :, 0].t()
      want = torch.stack([w[n + t] for w, n in zip(whole, lengths)])
      tol = 64 * max(torch.finfo(dtype).eps / 2, 2.0 ** -20) * want.abs().max().item()
      assert (got.double() - want.double()).abs().max().item() <= tol
  with pytest.raises(RuntimeError, match='causal'):
    ocnn.OctreeAttention(32, 4).cuda().step(x, at, caches[0])


def test_modules_keep_their_frequencies():
  layer = ocnn.OctreeAttention(32, 2).cuda().half()
  assert layer.freqs.dtype == torch.float64 and layer.freqs.is_cuda
  assert torch.equal(layer.freqs.cpu(), ocnn.rotary_freqs(layer.sections, device='cpu'))
  assert 'freqs' not in layer.state_dict()
  for bad in ((30, 4, None), (32, 4, 3), (12, 4, 4)):
    with pytest.raises(ValueError):
      ocnn.OctreeAttention(*bad)


def test_no_forward_mode_derivatives():
  from torch.autograd import forward_ad
  q, w = randn(6, 2, 16), randn(16)
  cache = torch.zeros(6, 4, 2, 16, device='cuda')
  off, lengths = (torch.tensor(x, dtype=torch.int32, device='cuda') for x in ([0, 6], [0] * 6))
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(q, torch.ones_like(q))
    for call in (lambda: ocnn.octree_attention(q, dual, q, off), lambda: ocnn.add_rms_norm(q, dual, w),
                 lambda: ocnn.octree_attention_step(dual, q, q, cache, cache.clone(), lengths),
                 lambda: ocnn.octree_rotary(dual, q[:, 0, :3], ocnn.rotary_freqs([4, 2, 2]), [4, 2, 2])):
      with pytest.raises(RuntimeError, match='forward-mode'):
        call()


def test_block_under_autocast():
  """Products and attention in bfloat16, norms and the residual in float32: no more roundings than bfloat16 data has
  (test_block), so its bound holds."""
  torch.manual_seed(0)
  _, seq = a_level(4)
  block = ocnn.OctreeAttentionBlock(64, 4, kv_heads=2, window=40, sinks=1).cuda()
  data = randn(1, 64, seq.positions.shape[0], 1).contiguous(memory_format=torch.channels_last)
  want = block_reference(block, data, seq, None)
  leaf = data.clone().requires_grad_()
  with torch.autocast('cuda', dtype=BF16):
    out = block(leaf, seq)
  assert out.dtype == F32
  assert (out[0, :, :, 0].t().double() - want).abs().max().item() <= 32 * 2.0 ** -8 * want.abs().max().item()
  out.sum().backward()
  assert leaf.grad.dtype == F32 and all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())
