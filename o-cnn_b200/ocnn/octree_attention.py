"""Attention over octree nodes: a layer that mixes a node with the nodes around it, as OctreeConv does, but with
weights formed from the data and a reach that is not bound to 27 cells.

A level's nodes lie shape by shape in Morton order, so a window of consecutive nodes is a neighbourhood in space.
`octree_sequence` says where each shape of a batch begins and where its nodes are; `octree_attention` lets a node see
a window of its shape's nodes and, if wanted, the shape's first ones; `octree_rotary` turns the channels of queries and
keys by the nodes' positions, so that their products depend on where nodes stand to each other; `add_rms_norm` is the
norm between the layers, with the residual's addition.  `OctreeAttention` and `OctreeAttentionBlock` put them together, and
`octree_attention_step` serves networks that produce a shape node by node.

The functions take rows of heads, [n, heads, dim], in float32, bfloat16 or float16, with any strides whose last is 1 (a
slice of one product for queries, keys and values needs no copy).  The modules take and return node data [1, C, H, 1].
"""
import collections

import torch
from torch import nn as _nn

from . import nn
from .modules import OctreeConv1x1, _stock_conv1x1, hooked

OctreeSequence = collections.namedtuple('OctreeSequence', ['offsets', 'positions'])
OctreeSequence.__doc__ = """The nodes of a level as sequences, one per shape: `offsets` int32 [batch + 1], and the cell
of every node, `positions` float32 [n, 3]."""


def octree_sequence(octree, depth, nempty=False):
  """The OctreeSequence of a level's nodes (of its non-empty ones when nempty).  It serves every layer of the level."""
  info = nn.octree_info(octree)
  batch = info[1]
  xyz = nn.octree_decode_key(nn.octree_property(octree, 'xyz', depth)).float()
  if nempty:
    xyz = nn.octree_depad(xyz.t().contiguous().view(1, 4, -1, 1), octree, depth).view(4, -1).t()
  shapes = torch.arange(batch + 1, device=xyz.device, dtype=torch.float32)
  offsets = torch.searchsorted(xyz[:, 3].contiguous(), shapes, out_int32=True)
  return OctreeSequence(offsets, xyz[:, :3].contiguous())


def rotary_freqs(sections, base=100.0, device='cuda'):
  """Radians per cell for `octree_rotary`: an axis that turns n pairs of channels has base ** (-i / n), i < n."""
  freqs = [base ** (-i / n) for n in sections for i in range(n)]
  return torch.tensor(freqs, dtype=torch.float64, device=device)


def octree_rotary(data, positions, freqs, sections, interleaved=False):
  """Channels of every head turned in pairs: pair t of node i by the angle positions[i, axis of t] * freqs[t].

  data [n, heads, dim]; positions [n, axes] int32 or float32; freqs [pairs] float64 (`rotary_freqs`); sections: pairs per
  axis, dim / 2 in all at most (the others pass through).  Pairs are channels (t, t + dim / 2), or (2t, 2t + 1) when
  interleaved.  Differentiable in data, once."""
  return nn.octree_rotary(data, positions, freqs, list(sections), interleaved)


def add_rms_norm(data, residual, weight, eps=1e-6):
  """(norm, sum): sum = data + residual, norm = sum / sqrt(mean(sum ** 2) + eps) * weight over the last dimension.

  residual None: sum is data itself.  weight: float32, or of the data's type.  Differentiable, once."""
  return tuple(nn.add_rms_norm(data, residual, weight, eps))


def octree_attention(q, k, v, offsets, window=0, sinks=0, causal=False, mask=None, scale=None):
  """Attention of every node over a window of its sequence and the sequence's first nodes.

  q [n, heads, dim], k and v [n, key heads, dim] (heads a multiple of key heads; dim up to 128); offsets int32
  [batch + 1], ascending: sequence b holds the nodes offsets[b] .. offsets[b + 1] - 1.  Node i sees key j of its
  sequence when |i - j| < window (window 0: always) or j is one of the first `sinks` (up to 64); causal: and j <= i;
  mask (bool [n]): and mask[j].  scale: 1 / sqrt(dim) unless given.  A node that sees nothing, or that is in no
  sequence, has a row of zeros.  Differentiable in q, k and v, once; the gradients are the same bits every time."""
  return nn.octree_attention(q, k, v, offsets, window, sinks, causal, mask, scale)


def octree_attention_step(q, k, v, k_cache, v_cache, lengths, window=0, sinks=0, scale=None):
  """Causal attention of one new node per sequence: k and v are written into the caches at position lengths[b] (int32,
  left as it is), and q sees that position and those before it, as in `octree_attention`.

  q [batch, heads, dim], k and v [batch, key heads, dim], caches [batch, capacity, key heads, dim]; rows of a
  multiple of 16 bytes.  Position x is kept at place x of a cache; where window + sinks <= capacity, those behind the first
  `sinks` take turns (place sinks + (x - sinks) % (capacity - sinks)) and a sequence may grow without end, otherwise one
  that has outgrown its cache is left as it is and its output is NaN.  A negative length: the sequence is passed over, its
  output zero.  No gradient."""
  return nn.octree_attention_step(q, k, v, k_cache, v_cache, lengths, window, sinks, scale)


class AddRMSNorm(_nn.Module):
  """`add_rms_norm` on node data [1, C, H, 1]: forward(data, residual=None) -> (norm, sum), channels_last, in the wider of
  the two's types."""

  def __init__(self, channels, eps=1e-6):
    super().__init__()
    self.eps = eps
    self.weight = _nn.Parameter(torch.ones(channels))

  def forward(self, data, residual=None):
    if residual is not None and residual.dtype != data.dtype:    # (autocast: a 16-bit branch joins float32 data)
      dtype = torch.promote_types(data.dtype, residual.dtype)
      data, residual = data.to(dtype), residual.to(dtype)
    norm, total = add_rms_norm(_rows(data), None if residual is None else _rows(residual), self.weight, self.eps)
    return _nodes(norm), _nodes(total)

  def extra_repr(self):
    return 'channels={}, eps={}'.format(self.weight.shape[0], self.eps)


def _rows(data):
  """[1, C, H, 1] as rows [H, C]: a view of channels_last data."""
  assert data.dim() == 4 and data.size(0) == 1 and data.size(3) == 1
  return data[0, :, :, 0].t().contiguous()


def _nodes(rows):
  """Rows [H, C] as node data [1, C, H, 1], channels_last: a view."""
  return rows.view(1, rows.shape[0], 1, rows.shape[1]).permute(0, 3, 1, 2)


def _called(layer, data):
  """A layer whose product someone asked to see (hooks; a weight that a hook forms) or replaced: its own call."""
  autocast = torch.is_autocast_enabled('cuda')
  x = data
  if not autocast:                                       # (a Conv1d takes data of its parameters' type alone)
    x = data.to(next((p.dtype for p in layer.parameters()), data.dtype))
  out = layer(x) if type(layer) is not OctreeConv1x1 or hooked(layer) else layer.conv1x1(x.squeeze(-1)).unsqueeze(-1)
  return out if autocast else out.to(data.dtype)


def _linear(layer, data, residual=None, relu=False):
  """An OctreeConv1x1 on channels_last data, whose output is channels_last too, in the data's type (under autocast: in that
  one's, or the residual's)."""
  if type(layer) is not OctreeConv1x1 or not _stock_conv1x1(layer.conv1x1) or hooked(layer, layer.conv1x1):
    out = _called(layer, data)
    if residual is not None:
      out = out + residual
    out = torch.relu(out) if relu else out
    return out.contiguous(memory_format=torch.channels_last)
  conv = layer.conv1x1
  if data.shape[2] == 0 or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in
                                                           (data, conv.weight, conv.bias, residual)):
    rows = _rows(data)
    bias = None if conv.bias is None else conv.bias.to(rows.dtype)
    out = _nodes(torch.nn.functional.linear(rows, conv.weight[:, :, 0].to(rows.dtype), bias))
    if residual is not None:
      out = out + residual
    return torch.relu(out) if relu else out
  if torch.is_autocast_enabled('cuda'):                  # (as torch's linear does above)
    data = data.to(torch.get_autocast_dtype('cuda'))
  if residual is None or residual.dtype == data.dtype:
    return layer.run(data, residual=residual, relu=relu)
  out = layer.run(data) + residual
  return torch.relu(out) if relu else out


class AttentionCache:
  """What `OctreeAttention.step` keeps of a layer's nodes: keys and values [batch, capacity, key heads, dim], and how many
  nodes each sequence has (`lengths`; set one to -1 to pass a sequence over)."""

  def __init__(self, batch, capacity, kv_heads, dim, dtype=torch.bfloat16, device='cuda'):
    self.k = torch.zeros(batch, capacity, kv_heads, dim, dtype=dtype, device=device)
    self.v = torch.zeros_like(self.k)
    self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)

  def fill(self, k, v, offsets, sinks=0):
    """The nodes of a packed batch (as in `octree_attention`), as many of each sequence as `step` will look at: all, or
    the first `sinks` and the last capacity - sinks."""
    capacity = self.k.shape[1]
    if offsets.shape[0] != self.lengths.shape[0] + 1:
      raise RuntimeError('AttentionCache.fill: {} sequences for a cache of {}'.format(offsets.shape[0] - 1, self.lengths.shape[0]))
    node = torch.arange(k.shape[0], device=k.device)
    ends = offsets.long()
    b = torch.searchsorted(ends, node, right=True) - 1
    inside = (b >= 0) & (b < ends.shape[0] - 1)
    b = b.clamp(0, ends.shape[0] - 2)
    at, left = node - ends[b], ends[b + 1] - node
    keep = inside & ((at < sinks) | (left <= capacity - sinks))
    place = torch.where(at < capacity, at, sinks + (at - sinks) % max(capacity - sinks, 1))
    keep &= place < capacity                 # (more first nodes than places: what does not fit has none)
    b, place = b[keep], place[keep]
    self.k[b, place], self.v[b, place] = self.typed(k[keep].detach(), v[keep].detach())
    self.lengths.copy_(ends[1:] - ends[:-1])

  def typed(self, *rows):
    """Rows as autocast's products give them, in the cache's type."""
    return [x.to(self.k.dtype) for x in rows] if torch.is_autocast_enabled('cuda') else rows


class OctreeAttention(_nn.Module):
  """Queries, keys and values of every node by a 1x1 layer, rotary positions by its cell, attention over a window of its
  shape's nodes, and a 1x1 layer behind it (with the residual's addition in its epilogue when one is given)."""

  def __init__(self, channels, heads, kv_heads=None, window=128, sinks=0, causal=False, base=100.0):
    super().__init__()
    kv_heads = heads if kv_heads is None else kv_heads
    if channels % heads or (channels // heads) % 2 or heads % kv_heads:
      raise ValueError('{} channels in {} heads over {} key heads'.format(channels, heads, kv_heads))
    self.channels, self.heads, self.kv_heads = channels, heads, kv_heads
    self.window, self.sinks, self.causal = window, sinks, causal
    self.dim = channels // heads
    third = self.dim // 6
    self.sections = [self.dim // 2 - 2 * third, third, third]
    self.qkv = OctreeConv1x1(channels, (heads + 2 * kv_heads) * self.dim)
    self.proj = OctreeConv1x1(heads * self.dim, channels)
    self.register_buffer('freqs', rotary_freqs(self.sections, base, 'cpu'), persistent=False)

  def _apply(self, fn, *args, **kwargs):
    freqs = self.freqs
    super()._apply(fn, *args, **kwargs)
    # (.half() and the like are for the weights: the frequencies stay in 64 bits, as they were made)
    if self.freqs.dtype != torch.float64:
      self.freqs = freqs.to(self.freqs.device)
    return self

  def _heads(self, data, positions):
    """Rotated queries and keys, and values: [H, heads, dim] each."""
    turned = self.heads + self.kv_heads
    rows = _rows(_linear(self.qkv, data)).view(-1, turned + self.kv_heads, self.dim)
    qk = octree_rotary(rows[:, :turned], positions, self.freqs, self.sections)
    return qk[:, :self.heads], qk[:, self.heads:], rows[:, turned:]

  def forward(self, data, sequence, mask=None, residual=None, cache=None):
    """data [1, C, H, 1]; sequence: `octree_sequence` of its level.  cache: an AttentionCache to fill for `step`, which sees
    every node of it: not beside a mask."""
    if mask is not None and cache is not None:
      raise RuntimeError('OctreeAttention: a step would see the nodes that the mask hides (a cache beside a mask)')
    q, k, v = self._heads(data.contiguous(memory_format=torch.channels_last), sequence.positions)
    out = octree_attention(q, k, v, sequence.offsets, self.window, self.sinks, self.causal, mask)
    if cache is not None:
      cache.fill(k, v, sequence.offsets, self.sinks)
    return _linear(self.proj, _nodes(out.flatten(1)), residual)

  def step(self, data, positions, cache, residual=None):
    """One new node per sequence: data [1, C, batch, 1], their cells [batch, 3].  The cache takes them in."""
    if not self.causal:
      raise RuntimeError('OctreeAttention.step: only a causal layer can be run node by node')
    with torch.no_grad():
      q, k, v = self._heads(data.contiguous(memory_format=torch.channels_last), positions)
      q, k, v = cache.typed(q, k, v)
      out = octree_attention_step(q, k, v, cache.k, cache.v, cache.lengths, self.window, self.sinks)
      cache.lengths += (cache.lengths >= 0).to(torch.int32)
      return _linear(self.proj, _nodes(out.flatten(1)), residual)

  def extra_repr(self):
    return 'channels={}, heads={}, kv_heads={}, window={}, sinks={}, causal={}'.format(
        self.channels, self.heads, self.kv_heads, self.window, self.sinks, self.causal)


class OctreeAttentionBlock(_nn.Module):
  """Norm, attention, residual and norm, two 1x1 layers with a ReLU between them, residual."""

  def __init__(self, channels, heads, kv_heads=None, window=128, sinks=0, causal=False, ratio=4, base=100.0):
    super().__init__()
    self.norm1, self.norm2 = AddRMSNorm(channels), AddRMSNorm(channels)
    self.attention = OctreeAttention(channels, heads, kv_heads, window, sinks, causal, base)
    self.fc1 = OctreeConv1x1(channels, ratio * channels, use_bias=True)
    self.fc2 = OctreeConv1x1(ratio * channels, channels, use_bias=True)

  def _mlp(self, branch, data):
    norm, total = self.norm2(branch, data)
    return _linear(self.fc2, _linear(self.fc1, norm, relu=True), total)

  def forward(self, data, sequence, mask=None, cache=None):
    data = data.contiguous(memory_format=torch.channels_last)
    return self._mlp(self.attention(self.norm1(data)[0], sequence, mask, cache=cache), data)

  def step(self, data, positions, cache):
    with torch.no_grad():
      data = data.contiguous(memory_format=torch.channels_last)
      return self._mlp(self.attention.step(self.norm1(data)[0], positions, cache), data)
