"""What the C entry points of the attention layer refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch

import ocnn

L = ctypes.CDLL(ocnn.LIBRARY)
L.ocnn_last_error.restype = ctypes.c_char_p
L.ocnn_octree_attention_backward_workspace_bytes.restype = ctypes.c_size_t
OK, INVALID, UNSUPPORTED, CAPACITY = 0, 1, 2, 4
I64, I32, P = ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p


class Attention(ctypes.Structure):
  _fields_ = [('q', P), ('k', P), ('v', P), ('qs', I64 * 2), ('ks', I64 * 2), ('vs', I64 * 2), ('offsets', P), ('mask', P)] + \
      [(n, I32) for n in ('batch', 'n', 'heads', 'kv_heads', 'dim', 'window', 'sinks', 'causal', 'dtype')] + \
      [('scale', ctypes.c_float)]


class Cache(ctypes.Structure):
  _fields_ = [('k', P), ('v', P), ('ks', I64 * 3), ('vs', I64 * 3), ('lengths', P)] + \
      [(n, I32) for n in ('batch', 'capacity', 'kv_heads', 'dim', 'dtype')]


def attention(**kw):
  a = Attention(q=64, k=64, v=64, offsets=64, batch=1, n=8, heads=4, kv_heads=2, dim=32, dtype=1, scale=1.0)
  for name, value in kw.items():
    setattr(a, name, value)
  return a


@pytest.mark.parametrize('kw,status', [(dict(n=-1), INVALID), (dict(heads=0), INVALID), (dict(heads=3), INVALID),
                                       (dict(dim=0), INVALID), (dict(dtype=3), INVALID), (dict(window=-1), INVALID),
                                       (dict(sinks=-2), INVALID), (dict(q=None), INVALID), (dict(offsets=None), INVALID),
                                       (dict(dim=136), UNSUPPORTED), (dict(sinks=65), UNSUPPORTED), (dict(n=0), OK)])
def test_attention(kw, status):
  a = attention(**kw)
  assert L.ocnn_octree_attention(ctypes.byref(a), P(64), None, P(64), None) == status
  grad = (I64 * 2)(128, 32)
  assert L.ocnn_octree_attention_backward(ctypes.byref(a), P(64), P(64), P(64), grad, P(64), P(64), P(64), P(64),
                                          ctypes.c_size_t(1 << 40), P(64), None) == status
  if status != OK:
    assert b'ocnn_octree_attention' in L.ocnn_last_error()


def test_attention_workspace():
  a = attention(n=5000, batch=3, sinks=4, window=16)
  need = L.ocnn_octree_attention_backward_workspace_bytes(ctypes.byref(a))
  assert need >= 4 * 5000 * 4 + (20 + 3) * 2 * 4 * 2 * 32 * 4
  grad = (I64 * 2)(128, 32)
  assert L.ocnn_octree_attention_backward(ctypes.byref(a), P(64), P(64), P(64), grad, P(64), P(64), P(64), P(64),
                                          ctypes.c_size_t(need - 1), P(64), None) == CAPACITY
  assert L.ocnn_octree_attention(ctypes.byref(a), None, None, P(64), None) == INVALID


@pytest.mark.parametrize('kw,heads,window,status', [
    (dict(capacity=0), 4, 0, INVALID), (dict(dtype=7), 4, 0, INVALID), ({}, 3, 0, INVALID), ({}, 4, -1, INVALID),
    (dict(dim=136), 4, 0, UNSUPPORTED), (dict(dim=12), 4, 0, UNSUPPORTED), (dict(lengths=None), 4, 0, INVALID),
    (dict(k=8), 4, 0, INVALID), (dict(batch=0), 4, 0, OK)])
def test_step(kw, heads, window, status):
  c = Cache(k=64, v=64, ks=(I64 * 3)(2048, 64, 32), vs=(I64 * 3)(2048, 64, 32), lengths=64, batch=2, capacity=32,
            kv_heads=2, dim=32, dtype=1)
  for name, value in kw.items():
    setattr(c, name, value)
  s = (I64 * 2)(128, 32)
  assert L.ocnn_octree_attention_step(ctypes.byref(c), P(64), s, P(64), s, P(64), s, P(64), heads, window, 0,
                                      ctypes.c_float(1.0), None) == status


def test_rotary_and_norm():
  s = (I64 * 2)(64, 16)

  def rotary(dim=16, axes=2, sections=(4, 4), rows=5, dtype=0, x=64):
    return L.ocnn_octree_rotary(P(x), s, P(64), P(64), 0, P(64), axes, (ctypes.c_int * len(sections))(*sections),
                                I64(rows), 4, dim, 0, 0, dtype, None)
  assert [rotary(dim=15), rotary(sections=(5, 4)), rotary(sections=(-1, 4)), rotary(axes=0), rotary(axes=9, sections=(0,) * 9),
          rotary(dtype=5), rotary(x=None)] == [INVALID] * 7
  assert rotary(dim=1024) == UNSUPPORTED and rotary(rows=0) == OK

  def norm(channels=16, weight_dtype=0, rows=5, dtype=1, x=64):
    return L.ocnn_add_rms_norm(P(x), I64(16), None, I64(0), P(64), weight_dtype, None, P(64), I64(rows), channels,
                               ctypes.c_float(1e-6), dtype, None)
  assert [norm(channels=0), norm(weight_dtype=2), norm(dtype=9), norm(rows=-1), norm(x=None)] == [INVALID] * 5
  assert norm(rows=0) == OK
  assert L.ocnn_add_rms_norm_backward(P(64), I64(16), None, I64(0), P(64), 0, None, I64(0), None, I64(0), P(64), P(64), I64(5), 16,
                                      ctypes.c_float(1e-6), 1, None, ctypes.c_size_t(0), None) == CAPACITY


def test_no_cpu_path():
  x = torch.zeros(4, 2, 16)
  off = torch.zeros(2, dtype=torch.int32)
  for call in (lambda: ocnn.octree_attention(x, x, x, off),
               lambda: ocnn.octree_attention_step(x, x, x, x[None], x[None], off),
               lambda: ocnn.octree_rotary(x, torch.zeros(4, 1, dtype=torch.int32), ocnn.rotary_freqs([2], device='cpu'), [2]),
               lambda: ocnn.add_rms_norm(x, None, torch.ones(16))):
    with pytest.raises(RuntimeError, match='CUDA'):
      call()


def test_attention_of_too_many_sequences():
  a = attention(batch=(1 << 24) + 1)
  assert L.ocnn_octree_attention(ctypes.byref(a), P(64), None, P(64), None) == UNSUPPORTED
  assert L.ocnn_octree_attention_backward_workspace_bytes(ctypes.byref(a)) == 0
