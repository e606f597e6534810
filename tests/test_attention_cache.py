"""The attention layer's cache and its refusals, on the CPU."""
import pytest
import torch

import ocnn


def filled(lengths, capacity, sinks, first=0, tail=0):
  """(cache, packed keys): key of node t of sequence b is 1000 b + t + 1."""
  cache = ocnn.AttentionCache(len(lengths), capacity, 1, 8, torch.float32, 'cpu')
  keys = torch.cat([torch.zeros(first)] + [1000.0 * b + 1 + torch.arange(float(n)) for b, n in enumerate(lengths)] +
                   [torch.zeros(tail)])
  rows = keys[:, None, None].expand(-1, 1, 8)
  offsets = torch.tensor([first + sum(lengths[:b]) for b in range(len(lengths) + 1)], dtype=torch.int32)
  cache.fill(rows, -rows, offsets, sinks)
  return cache


@pytest.mark.parametrize('capacity,sinks', [(1, 0), (2, 4), (4, 4), (3, 5), (8, 3), (8, 0), (16, 64)])
def test_fill(capacity, sinks):
  """Every position that a place is for lies there, the last that came to it; more first nodes than the cache has room for are
  a cache that does not roll: as many positions as it holds."""
  lengths = [0, 1, capacity, capacity + 1, 3 * capacity + 2]
  cache = filled(lengths, capacity, sinks, first=2, tail=3)
  assert cache.lengths.tolist() == lengths
  for b, n in enumerate(lengths):
    places = {}
    for x in range(n):
      place = x if x < capacity else sinks + (x - sinks) % (capacity - sinks) if sinks < capacity else None
      if place is not None:
        places[place] = 1000 * b + x + 1
    got = cache.k[b, :, 0, 0]
    assert got.tolist() == [float(places.get(place, 0)) for place in range(capacity)], (b, n)
    assert torch.equal(cache.v[b], -cache.k[b])


def test_fill_of_another_batch():
  for sequences in (1, 2, 4):
    cache = ocnn.AttentionCache(3, 8, 1, 8, torch.float32, 'cpu')
    offsets = torch.arange(sequences + 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match='sequences'):
      cache.fill(torch.zeros(sequences, 1, 8), torch.zeros(sequences, 1, 8), offsets)
    assert not cache.lengths.any()


def test_fill_of_no_sequences():
  cache = ocnn.AttentionCache(0, 8, 1, 8, torch.float32, 'cpu')
  cache.fill(torch.zeros(2, 1, 8), torch.zeros(2, 1, 8), torch.zeros(1, dtype=torch.int32))
  assert cache.lengths.shape == (0,)


def test_no_mask_beside_a_cache():
  """A step cannot know which of the cache's nodes were hidden."""
  cache = ocnn.AttentionCache(1, 8, 4, 8, torch.float32, 'cpu')
  data, mask = torch.zeros(1, 32, 5, 1), torch.ones(5, dtype=torch.bool)
  seq = ocnn.OctreeSequence(torch.tensor([0, 5], dtype=torch.int32), torch.zeros(5, 3))
  with pytest.raises(RuntimeError, match='mask'):
    ocnn.OctreeAttention(32, 4, causal=True)(data, seq, mask, cache=cache)


def test_tracing_is_refused():
  """A recording would hold none of the kernels' work."""
  x, off = torch.zeros(4, 2, 16), torch.tensor([0, 4], dtype=torch.int32)
  pos, freqs = torch.zeros(4, 1, dtype=torch.int32), ocnn.rotary_freqs([2], device='cpu')
  for call in (lambda x: ocnn.octree_attention(x, x, x, off), lambda x: ocnn.octree_rotary(x, pos, freqs, [2]),
               lambda x: ocnn.add_rms_norm(x, None, torch.ones(16)),
               lambda x: ocnn.octree_attention_step(x, x, x, x[:, None], x[:, None], torch.zeros(4, dtype=torch.int32))):
    with pytest.raises(RuntimeError, match='traced'):
      torch.jit.trace(call, (x,), check_trace=False)


def test_transforms_are_refused():
  x, off = torch.zeros(4, 2, 16), torch.tensor([0, 4], dtype=torch.int32)
  pos, freqs = torch.zeros(4, 1, dtype=torch.int32), ocnn.rotary_freqs([2], device='cpu')
  calls = (lambda x: ocnn.octree_attention(x, x, x, off), lambda x: ocnn.octree_rotary(x, pos, freqs, [2]),
           lambda x: ocnn.add_rms_norm(x, None, torch.ones(16))[0])
  for call in calls:
    with pytest.raises(RuntimeError, match='torch.func'):
      torch.func.grad(lambda x: call(x).sum())(x)
    with pytest.raises(RuntimeError, match='torch.func'):
      torch.vmap(call)(x[None])


def test_workspace_of_many_short_sequences():
  """Slots for sums from far are made for sequences that can have them: those longer than the window."""
  import ctypes
  import test_attention_host as host
  need = host.L.ocnn_octree_attention_backward_workspace_bytes
  slot = 4 * 16 * 2 * 64 * 4                                              # key heads, first nodes, dK and dV, fp32
  rest = (1000000 // 256 + 64 + 8 * 1000000) * 4
  a = dict(n=1000000, heads=8, kv_heads=4, dim=64, sinks=16)
  many = need(ctypes.byref(host.attention(batch=100000, window=1000, **a)))
  assert many <= rest + (1000000 // 256 + 1000000 // 1001 + 2) * slot
  few = need(ctypes.byref(host.attention(batch=10, window=1000, **a)))
  assert (1000000 // 256) * slot <= few <= rest + (1000000 // 256 + 1 + 10) * slot


def test_too_many_sequences_or_heads():
  """The message says what is too many."""
  import ctypes
  import test_attention_host as host
  cache = host.Cache(k=64, v=64, ks=(host.I64 * 3)(2048, 64, 32), vs=(host.I64 * 3)(2048, 64, 32), lengths=64, batch=65536,
                     capacity=32, kv_heads=2, dim=32, dtype=1)
  s, p = (host.I64 * 2)(128, 32), host.P(64)
  step = lambda heads: host.L.ocnn_octree_attention_step(ctypes.byref(cache), p, s, p, s, p, s, p, heads, 0, 0,
                                                         ctypes.c_float(1.0), None)
  assert step(4) == host.UNSUPPORTED and b'65536 sequences, 4 heads' in host.L.ocnn_last_error()
  cache.batch = 2
  assert step(65536) == host.UNSUPPORTED and b'2 sequences, 65536 heads' in host.L.ocnn_last_error()
  a = host.attention(heads=65536, kv_heads=1)
  assert host.L.ocnn_octree_attention(ctypes.byref(a), p, None, p, None) == host.UNSUPPORTED
  assert b'65536 heads' in host.L.ocnn_last_error()


def test_gradients_of_keys_without_those_of_values():
  import ctypes
  import test_attention_host as host
  a, p, s = host.attention(), host.P(64), (host.I64 * 2)(128, 32)
  call = lambda dq, dk, dv: host.L.ocnn_octree_attention_backward(ctypes.byref(a), p, p, p, s, dq, dk, dv, p, ctypes.c_size_t(0), p,
                                                                  None)
  assert [call(p, None, p), call(p, p, None), call(None, p, p)] == [host.INVALID] * 3
  assert call(p, None, None) == host.CAPACITY
