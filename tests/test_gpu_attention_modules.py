"""The attention layer's modules as a network uses them: hooks and replaced layers, autocast, empty levels, caches."""
import sys

import pytest
import torch

import ocnn

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def nodes(n, channels, dtype=F32, seed=0):
  x = torch.randn(n, channels, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda').to(dtype)
  return x[None, :, None].permute(0, 3, 1, 2)


def sequence(lengths):
  offsets = torch.tensor([0] + [sum(lengths[:i + 1]) for i in range(len(lengths))], dtype=torch.int32, device='cuda')
  gen = torch.Generator(device='cuda').manual_seed(9)
  return ocnn.OctreeSequence(offsets, torch.randint(0, 32, (sum(lengths), 3), generator=gen, device='cuda').float())


def block(**kw):
  torch.manual_seed(0)
  return ocnn.OctreeAttentionBlock(32, 4, kv_heads=2, window=12, sinks=1, **kw).cuda()


# ---- hooks and replaced layers ------------------------------------------------------------------------------------------
LAYERS = ('attention.qkv', 'attention.proj', 'fc1', 'fc2')


@pytest.mark.parametrize('inner', [False, True])
def test_hooks_see_the_layers(inner):
  """Forward hooks on the 1x1 layers and on the Conv1d that holds their weights run, in training, and what one returns is
  what goes on; without gradients the layers' own are run."""
  net, x, seq = block(), nodes(50, 32), sequence([30, 20])
  want = net(x, seq)
  seen = []
  for name in LAYERS:
    layer = net.get_submodule(name)
    (layer.conv1x1 if inner else layer).register_forward_hook(lambda m, i, o, name=name: seen.append(name))
  got = net(x, seq)
  tol = 32 * 2.0 ** -11 * want.abs().max()         # (a Conv1d may take its products in TF32)
  assert seen == list(LAYERS) and (got - want).abs().max() <= tol
  got.sum().backward()
  assert all(p.grad is not None for p in net.parameters())
  del seen[:]
  with torch.no_grad():
    assert (net(x, seq) - want).abs().max() <= tol and seen == list(LAYERS)
  net.fc2.register_forward_hook(lambda m, i, o: torch.zeros_like(o))
  assert (net(x, seq) - (x + net.attention(net.norm1(x)[0], seq))).abs().max() <= tol


def test_reparametrised_weights():
  """A weight that a forward-pre-hook forms from others is formed for every call; 16-bit data too."""
  net, x, seq = block(), nodes(50, 32), sequence([30, 20])
  with pytest.warns(FutureWarning):
    torch.nn.utils.weight_norm(net.attention.proj.conv1x1)
  plain = block()
  for grad in (True, False):
    for dtype, tol in ((F32, 32 * 2.0 ** -11), (BF16, 32 * 2.0 ** -8)):
      with torch.no_grad():
        net.attention.proj.conv1x1.weight_g.mul_(1.5)
        plain.attention.proj.conv1x1.weight.mul_(1.5)
      with torch.set_grad_enabled(grad):
        got, want = net(x.to(dtype), seq), plain(x.to(dtype), seq)
      assert got.dtype == dtype and (got - want).abs().max() <= tol * want.abs().max()


class Adapter(torch.nn.Module):
  """A Conv1d and a narrow branch beside it, without a weight of its own."""

  def __init__(self, base):
    super().__init__()
    self.base = base
    self.down = torch.nn.Conv1d(base.in_channels, 2, 1, bias=False).cuda()
    self.up = torch.nn.Conv1d(2, base.out_channels, 1, bias=False).cuda()

  def forward(self, x):
    return self.base(x) + self.up(self.down(x))


@pytest.mark.parametrize('autocast', [False, True])
def test_a_replaced_product(autocast):
  net, x, seq = block(), nodes(50, 32), sequence([30, 20])
  plain = block()
  adapter = net.fc1.conv1x1 = Adapter(net.fc1.conv1x1)
  with torch.no_grad():
    plain.fc1.conv1x1.weight += (adapter.up.weight[:, :, 0] @ adapter.down.weight[:, :, 0])[:, :, None]
  with torch.autocast('cuda', dtype=BF16, enabled=autocast):
    got, want = net(x, seq), plain(x, seq)
    with torch.no_grad():
      quiet = net(x, seq)
  tol = 32 * (2.0 ** -8 if autocast else 2.0 ** -11)
  assert (got - want).abs().max() <= tol * want.abs().max() and (quiet - want).abs().max() <= tol * want.abs().max()
  got.sum().backward()
  assert adapter.up.weight.grad is not None and adapter.base.weight.grad is not None


def test_biases_alone_are_trained():
  net, x, seq = block(), nodes(50, 32), sequence([30, 20])
  for name, p in net.named_parameters():
    p.requires_grad_(name.endswith('bias'))
  out = net(x, seq)
  out.sum().backward()
  assert net.fc1.conv1x1.bias.grad.any() and torch.equal(net.fc2.conv1x1.bias.grad, torch.full((32,), 50.0, device='cuda'))


# ---- autocast -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [BF16, F16])
def test_autocast_without_gradients(dtype, monkeypatch):
  """As in training: products and attention in the 16-bit type, norms and the residual in the data's."""
  module = sys.modules['ocnn.octree_attention']
  net, x, seq = block(causal=True), nodes(50, 32), sequence([30, 20])
  types, plain = [], module.octree_attention
  monkeypatch.setattr(module, 'octree_attention', lambda q, *a, **kw: types.append(q.dtype) or plain(q, *a, **kw))
  with torch.autocast('cuda', dtype=dtype):
    want = net(x, seq)
    with torch.no_grad():
      for cache in [ocnn.AttentionCache(2, 40, 2, 8, t) for t in (dtype, F32)]:
        got = net(x, seq, cache=cache)
        assert net.step(nodes(2, 32), torch.zeros(2, 3, device='cuda'), cache).dtype == F32
  assert types == [dtype] * 3 and got.dtype == want.dtype == F32
  # (both are within 32 half steps of the definition: six roundings on the way)
  assert (got - want).abs().max().item() <= 64 * torch.finfo(dtype).eps / 2 * want.abs().max().item()


# ---- levels and batches of no or one node ---------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('n', [0, 1])
def test_hardly_any_nodes(n, dtype):
  net, seq = block(causal=True), sequence([0, n])
  leaf = nodes(n, 32, dtype).requires_grad_()
  out = net(leaf, seq)
  assert out.shape == (1, 32, n, 1) and out.dtype == dtype
  out.sum().backward()
  assert leaf.grad.shape == leaf.shape and all(bool(p.grad.any()) == bool(n) for p in net.parameters() if p.dim() < 3)
  with torch.no_grad():
    quiet = net(leaf, seq)
    assert quiet.shape == (1, 32, n, 1)
    # (both within 32 half steps of the definition)
    assert n == 0 or (quiet - out).abs().max() <= 64 * max(torch.finfo(dtype).eps / 2, 2.0 ** -20) * out.abs().max()
    cache = ocnn.AttentionCache(n, 16, 2, 8, dtype)
    assert net.step(leaf, torch.zeros(n, 3, device='cuda'), cache).shape == (1, 32, n, 1)
