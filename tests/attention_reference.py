"""The attention operators from their definitions in 64 bits, with how far a kernel's result may be off.

A kernel holds scores, statistics and sums in 32 bits; with 16-bit data it rounds probabilities p and score gradients ds to
the data's type before the second products, the forward result before it is read again, and every result once.  With u
half a step of the type (`finfo.eps / 2`) and e the relative error of a probability (a score is a sum of dim products:
(dim + 4) 2^-24 sum |q k| scale, and 2^-21 for the exponential and its sum) the bounds are, element by element,
    out:  u |out| + (u + e) sum_j p |v|
    dv:   u |dv| + sum_i (u + e) p |dO|
    ds:   (u + e) |ds| + p ((dim + 4) 2^-24 sum |dO v| + (u + 2^-20) sum |dO out|);  dq, dk: that times |k|, |q| scale
each with 2^-20 of the sum of absolute terms for the additions in 32 bits.  A value below the type's smallest normal number
(2^-14 in float16) is rounded to a multiple of its smallest one: off by half of that, t = tiny * eps / 2 (2^-25), whatever
its size.  t comes on top of every result, and t sum |factor| where p and ds are rounded."""
import math

import torch

ADD = 2.0 ** -20


def visible(n, offsets, window, sinks, causal, mask, device):
  """bool [n, n]: node i sees key j."""
  i, j = torch.arange(n, device=device)[:, None], torch.arange(n, device=device)[None]
  out = torch.zeros(n, n, dtype=torch.bool, device=device)
  for s, e in zip(offsets[:-1], offsets[1:]):
    near = (i - j).abs() < window if window else torch.ones_like(out)
    see = (near | (j - s < sinks)) & (i >= s) & (i < e) & (j >= s) & (j < e)
    out |= see & (j <= i) if causal else see
  return out if mask is None else out & mask[None]


def attention(q, k, v, see, scale=None, grad=None):
  """{name: (value, bound)} in float64 for out and, with grad, dq, dk, dv."""
  u = torch.finfo(q.dtype).eps / 2
  t = torch.finfo(q.dtype).tiny * u
  n, heads, dim = q.shape
  kv, group = k.shape[1], q.shape[1] // k.shape[1]
  scale = 1 / math.sqrt(dim) if scale is None else scale
  clean = lambda x: x.detach().double().transpose(0, 1)
  q, k, v = clean(q), clean(k).repeat_interleave(group, 0), clean(v).repeat_interleave(group, 0)
  s = (q @ k.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
  p = torch.softmax(s, 2).nan_to_num(0.0)
  half = (dim + 4) * 2.0 ** -24
  e = (half * abs(scale) * (q.abs() @ k.abs().transpose(1, 2))).masked_fill(~see, 0).amax(2, keepdim=True) + 2.0 ** -21
  out = p @ v
  # (p is rounded before it is divided by its row's sum, which is 1 at least)
  seen, least = see.double(), t * (see.any(1).double())[None, :, None]
  heavy = p @ v.abs()
  back = lambda x: x.transpose(0, 1)
  res = {'out': (back(out), back(u * out.abs() + (u + e + ADD) * heavy + least + t * (seen @ v.abs())))}
  if grad is None:
    return res
  g = clean(grad)
  shared = lambda x: back(x.unflatten(0, (kv, group)).sum(1))
  dv, heavy = p.transpose(1, 2) @ g, ((u + e + ADD) * p).transpose(1, 2) @ g.abs()
  res['dv'] = shared(dv), u * shared(dv).abs() + shared(heavy + t * (seen.t() @ g.abs())) + t
  dp = g @ v.transpose(1, 2)
  delta = (g * out).sum(2, keepdim=True)
  ds = p * (dp - delta)
  off = (u + e + ADD) * ds.abs() + p * (half * (g.abs() @ v.abs().transpose(1, 2)) +
                                        (u + ADD) * (g * out).abs().sum(2, keepdim=True))
  dq = scale * (ds @ k)
  res['dq'] = back(dq), back(u * dq.abs() + abs(scale) * ((off + t * seen) @ k.abs()) + t)
  dk = shared(scale * (ds.transpose(1, 2) @ q))
  res['dk'] = dk, u * dk.abs() + shared(abs(scale) * ((off + t * seen).transpose(1, 2) @ q.abs())) + t
  return res


def check(got, want, what):
  value, bound = want
  off = (got.detach().double() - value).abs()
  worst = (off / (bound + 1e-30)).max().item() if off.numel() else 0.0
  assert bool((off <= bound + 1e-30).all()), '%s: %.3g of its bound, largest error %.3g' % (what, worst, off.max().item())
