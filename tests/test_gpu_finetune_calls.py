"""Blocks, attentions and maps that know nothing of the fine-tuning options: custom modules in the maps' places, subclasses
whose methods have no arguments for the options, and hooks on the maps.  Without an option in use they are called as
if there were none; a hook that returns a new input leaves the options of the call alone."""
import pytest
import torch
import torch.nn as nn

import flash_eq as fe

pytestmark = pytest.mark.gpu

LV = [0, 1, 2]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rel(a, b):
    return ((a.detach().double() - b.detach().double()).abs().max() / b.detach().double().abs().max()).item()


def inputs(dev, n=40, k=6, mult=16, dtype=torch.float32):
    g = gen(3)
    x = torch.rand(n, 3, generator=g) * 5
    d = torch.cdist(x, x) + 1e6 * torch.eye(n)
    src = torch.topk(d, k, largest=False).indices.reshape(-1).to(dev)
    dst = torch.arange(n).repeat_interleave(k).to(dev)
    x = x.to(dev)
    v = x[src] - x[dst]
    (P,) = fe.WignerDBasis([fe.Repr(LV, mult)]).to(dev)(v)
    f = torch.randn(n, mult, 9, generator=g).to(dev)
    return P.to(dtype), P.to(dtype), f.to(dtype), v.norm(dim=1).to(dtype), fe.Graph(src, dst, n)


def block_of(dev, seed=0, cls=fe.EquivariantTransformerBlock, **kw):
    torch.manual_seed(seed)
    r = fe.Repr(LV, 16)
    return cls(r, r, num_heads=4, max_dist=4.0, layer_scale_init=0.5, **kw).to(dev)


class Wrapped(nn.Module):
    """A user's module around a map: one input."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, f):
        return self.inner(f)


class OldLinear(fe.EquivariantLinear):
    def fused_ok(self, f):
        return super().fused_ok(f)

    def forward_layout(self, f, in_cm, out_cm):
        return super().forward_layout(f, in_cm, out_cm)

    def forward(self, f):
        return super().forward(f)


class OldEdgeAttention(fe.EquivariantEdgeAttention):
    def attention_weights(self, Q, K, graph, distances=None):
        return super().attention_weights(Q, K, graph, distances)

    def node_attention_weights(self, qk, graph, distances=None, cm=False):
        return super().node_attention_weights(qk, graph, distances, cm)


class OldAttention(fe.EquivariantAttention):
    def forward(self, P, Q_basis, node_features, distances, graph, edge_features=None):
        return super().forward(P, Q_basis, node_features, distances, graph, edge_features)


class OldBlock(fe.EquivariantTransformerBlock):
    def forward(self, P, Q, node_features, distances, graph, edge_features=None):
        return super().forward(P, Q, node_features, distances, graph, edge_features)


def as_class(module, cls):
    module.__class__ = cls
    return module


@pytest.mark.parametrize("wrap", [nn.Sequential, Wrapped])
def test_custom_modules_in_place_of_the_maps(dev, wrap):
    args = inputs(dev)
    plain, custom = block_of(dev, use_gating=False), block_of(dev, use_gating=False)
    custom.mlp_up, custom.mlp_down = wrap(custom.mlp_up), wrap(custom.mlp_down)
    assert torch.equal(custom(*args), plain(*args))
    custom.mlp_up, custom.mlp_act, custom.mlp_down = nn.Identity(), nn.Identity(), nn.Identity()
    assert custom(*args).shape == args[2].shape


@pytest.mark.parametrize("use_gating", [False, True])
@pytest.mark.parametrize("drop_path", [0.0, 0.5])                 # with it the MLP's result leaves node-major
def test_maps_with_one_argument(dev, use_gating, drop_path):
    args = inputs(dev)
    plain, old = (block_of(dev, use_gating=use_gating, drop_path=drop_path).eval() for _ in range(2))
    for m in (old.mlp_up, old.mlp_down, old.attn.linear_qk):
        as_class(m, OldLinear)
    assert torch.equal(old(*args), plain(*args))
    wide = inputs(dev)
    old.attn.linear_qk.activation = plain.attn.linear_qk.activation = nn.SiLU()       # the node-major path of the attention
    assert torch.equal(old(*wide), plain(*wide))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("edges", [False, True])
def test_subclasses_without_the_options(dev, dtype, edges):
    P, Q, f, r, graph = inputs(dev, dtype=dtype)
    e = torch.randn(r.shape[0], 16, 9, generator=gen(4)).to(dev, dtype) if edges else None
    plain, old = block_of(dev).to(dtype), block_of(dev, cls=OldBlock).to(dtype)
    as_class(old.attn, OldAttention)
    as_class(old.attn.attention, OldEdgeAttention)
    assert torch.equal(old(P, Q, f, r, graph, e), plain(P, Q, f, r, graph, e))
    assert torch.equal(old.attn(P, Q, f, r, graph, e), plain.attn(P, Q, f, r, graph, e))


def test_edge_attention_without_buckets(dev):
    *_, r, graph = inputs(dev)
    g = gen(5)
    Q, K = (torch.randn(r.shape[0], 4, 8, generator=g).to(dev) for _ in range(2))
    V = torch.randn(r.shape[0], 8, 9, generator=g).to(dev)
    plain = fe.EquivariantEdgeAttention(4, 8, distance_decay_scale=2.0).to(dev)
    old = OldEdgeAttention(4, 8, distance_decay_scale=2.0).to(dev)
    assert torch.equal(old(Q, K, V, graph, r), plain(Q, K, V, graph, r))


@pytest.mark.parametrize("keep", [False, True])
def test_hooks_see_the_features_alone_and_keep_the_adapters(dev, keep):
    """A forward pre-hook's return replaces the positional arguments: with the plan among them it would be lost."""
    args = inputs(dev)
    block = block_of(dev, use_gating=False).eval()
    with torch.no_grad():
        for i, p in enumerate(fe.add_adapters(block, 3, 4)):
            p.copy_(0.3 * torch.randn(p.shape, generator=gen(10 + i)))
    ids = torch.randint(-1, 3, (40,), generator=gen(6)).to(dev)
    want, without = block(*args, adapters=ids), block(*args)
    assert rel(want, without) > 1e-3
    seen = []

    def hook(module, inputs):
        seen.append(len(inputs))
        return (inputs[0] * 1.0,) if keep else None
    for m in (block.mlp_up, block.mlp_down):
        m.register_forward_pre_hook(hook)
    assert torch.equal(block(*args, adapters=ids), want) and torch.equal(block(*args), without)
    assert seen == [1, 1, 1, 1]


def test_adapters_through_a_map_that_cannot_take_them_are_refused(dev):
    block = block_of(dev, use_gating=False)
    fe.add_adapters(block, 3, 4)
    block.mlp_up = Wrapped(block.mlp_up)
    with pytest.raises(TypeError, match="plan"):
        block(*inputs(dev), adapters=torch.zeros(40, dtype=torch.int64, device=dev))
