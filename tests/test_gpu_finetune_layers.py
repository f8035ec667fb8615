"""The fine-tuning operators in the layers and the model: each option against what it stands for, all of them
together as a training loop uses them, and the refusals of their entry points.

The layers around the operators are the framework's float32 ones, whose results two ways of computing the same agree to
1e-5 of the largest (the bound of the framework's other layer tests); a test states where it needs more."""
import pytest
import torch

import flash_eq as fe
from flash_eq.capture import capture_step

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rel(a, b):
    return ((a.detach().double() - b.detach().double()).abs().max() / b.detach().double().abs().max()).item()


def cloud(dev, seed, n=40, k=8):
    """Points, their nearest neighbours (src -> dst) and features of degrees 0 and 1."""
    g = gen(seed)
    x = torch.rand(n, 3, generator=g) * 6
    d = torch.cdist(x, x) + 1e6 * torch.eye(n)
    src = torch.topk(d, k, largest=False).indices.reshape(-1)
    dst = torch.arange(n).repeat_interleave(k)
    return x.to(dev), fe.Graph(src.to(dev), dst.to(dev), n), torch.randn(n, 8, 4, generator=g).to(dev)


def model_of(dev, seed=0, **kw):
    torch.manual_seed(seed)
    lv = [0, 1, 2]
    m = fe.EquivariantTransformer(fe.Repr([0, 1], 8), fe.Repr(lv, 16), fe.Repr([0, 1], 8), num_layers=2, num_heads=4, max_dist=4.0,
                                  layer_scale_init=0.5, **kw).to(dev)
    return m


def stir(params, seed=1, scale=0.3):
    """Small random values for parameters that begin as zeros."""
    g = gen(seed)
    with torch.no_grad():
        for p in params:
            p.copy_(scale * torch.randn(p.shape, generator=g))


def score(y):
    """A loss that the final norm does not make constant (the mean square of the results is 1)."""
    return (y.float() * torch.linspace(-1, 1, y.numel(), device=y.device).view(y.shape)).mean()


def biases(m):
    return [x.bias for x in m.modules() if isinstance(x, fe.EquivariantEdgeAttention)]


def test_zero_bias_and_new_adapters_change_nothing(dev):
    x, graph, f = cloud(dev, 1)
    plain, tuned = model_of(dev).eval(), model_of(dev, bias_buckets=12, counter_dropout=True, dropout=0.3, feature_dropout=0.3).eval()
    fe.add_adapters(tuned, 3, 4)
    ids = torch.randint(-1, 3, (40,), generator=gen(2)).to(dev)
    want = plain(x, f, graph)
    assert rel(tuned(x, f, graph, adapters=ids), want) < 1e-5
    assert rel(tuned(x, f, graph), want) < 1e-5                       # without ids the maps alone


def test_bias_of_a_linear_decay_is_the_decay(dev):
    """A bias that falls with the bucket's distance is the fixed decay at those distances."""
    g = gen(3)
    n, E, H = 30, 240, 4
    src, dst = (torch.randint(0, n, (E,), generator=g).to(dev) for _ in range(2))
    graph = fe.Graph(src, dst, n)
    dist = (torch.randint(0, 16, (E,), generator=g).float() / 2).to(dev)           # at the buckets' lower ends
    buckets = fe.DistanceBuckets(16, 0.0, 7.5).to(dev)(dist)
    assert torch.equal(buckets.float() / 2, dist)
    a = fe.EquivariantEdgeAttention(H, 8, bias_buckets=16).to(dev)
    b = fe.EquivariantEdgeAttention(H, 8, distance_decay_scale=3.0).to(dev)
    with torch.no_grad():
        a.bias.copy_((-torch.arange(16).float() / 2 / 3.0)[:, None].expand(16, H))
    Q, K = torch.randn(E, H, 8, generator=g).to(dev), torch.randn(E, H, 8, generator=g).to(dev)
    assert rel(a.attention_weights(Q, K, graph, None, buckets), b.attention_weights(Q, K, graph, dist)) < 1e-5
    V = torch.randn(E, 8, 4, generator=g).to(dev)
    assert rel(a(Q, K, V, graph, None, buckets), b(Q, K, V, graph, dist)) < 1e-5
    qk = torch.randn(n, 2 * H * 2, 4, generator=g).to(dev)
    assert rel(a.node_attention_weights(qk, graph, buckets=buckets), b.node_attention_weights(qk, graph, dist)) < 1e-5
    cm = qk.permute(2, 0, 1).contiguous()
    assert rel(a.node_attention_weights(cm, graph, None, True, buckets), b.node_attention_weights(qk, graph, dist)) < 1e-5


def merged(model, a):
    """A copy of the model whose maps hold adapter a."""
    import copy
    m = copy.deepcopy(model)
    with torch.no_grad():
        for linear in m.modules():
            if isinstance(linear, fe.EquivariantLinear):
                low = linear.adapters
                linear.weight += low.scale * (low.up[a] @ low.down[a]).reshape(linear.weight.shape)
    return m


def test_structures_of_a_batch_each_with_its_adapter(dev):
    """Two structures in one batch, each with its own adapter, and one with none, against each alone through merged maps."""
    model = model_of(dev, bias_buckets=12).eval()
    low = fe.add_adapters(model, 2, 4, alpha=2)
    stir(low)
    stir(biases(model), 5)
    parts = [cloud(dev, 10 + i, n) for i, n in enumerate((40, 25, 30))]
    x = torch.cat([p[0] for p in parts])
    f = torch.cat([p[2] for p in parts])
    at, starts = 0, []
    for p in parts:
        starts.append(at)
        at += p[1].num_nodes
    graph = fe.Graph(torch.cat([p[1].src + s for p, s in zip(parts, starts)]), torch.cat([p[1].dst + s for p, s in zip(parts, starts)]), at)
    ids = torch.cat([torch.full((p[1].num_nodes,), i, device=dev) for p, i in zip(parts, (1, -1, 0))])
    with torch.no_grad():
        y = model(x, f, graph, adapters=ids)
        for (px, pg, pf), s, a in zip(parts, starts, (1, None, 0)):
            alone = model if a is None else merged(model, a)
            assert rel(y[s:s + pg.num_nodes], alone(px, pf, pg)) < 1e-5
        order = torch.randperm(at, generator=gen(4)).to(dev)            # nodes of the structures in any order
        place = torch.argsort(order)
        mixed = fe.Graph(place[graph.src], place[graph.dst], at)
        assert rel(model(x[order], f[order], mixed, adapters=ids[order]), y[order]) < 1e-5


def test_equivariance_with_all_options(dev):
    """Rotated inputs give rotated outputs under the same masks: a dropout of components would not."""
    from scipy.spatial.transform import Rotation
    R = torch.tensor(Rotation.random(random_state=3).as_matrix(), dtype=torch.float32, device=dev)
    model = model_of(dev, bias_buckets=12, counter_dropout=True, dropout=0.2, feature_dropout=0.2).train()
    stir(fe.add_adapters(model, 3, 4))
    stir(biases(model), 6)
    x, graph, f = cloud(dev, 7)
    ids = torch.randint(-1, 3, (40,), generator=gen(8)).to(dev)
    order = [1, 2, 0]                                                   # (y, z, x)
    R1 = R[order][:, order]

    def turned(t):
        return torch.cat([t[..., :1], t[..., 1:] @ R1.T], -1)

    def run(x, f):
        torch.manual_seed(11)
        return model(x, f, graph, adapters=ids)
    y = run(x, f)
    torch.manual_seed(12)
    other = model(x, f, graph, adapters=ids)
    assert rel(other, y) > 1e-2                                          # masks matter
    got = run(x @ R.T, turned(f))
    assert rel(got, turned(y)) < 1e-4                      # the bound of the framework's equivariance tests


def training(dev, dtype=torch.float32, **kw):
    model = model_of(dev, bias_buckets=12, counter_dropout=True, dropout=0.2, feature_dropout=0.1, **kw)
    params = fe.add_adapters(model, 3, 4)
    stir(params)
    stir(biases(model), 6)
    model.to(dtype).train()
    x, graph, f = cloud(dev, 20)
    ids = torch.randint(-1, 3, (40,), generator=gen(9)).to(dev)
    return model, x.to(dtype), graph, f.to(dtype), ids


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("experts", [0, 3])
def test_training_step_reaches_every_parameter(dev, dtype, experts):
    model, x, graph, f, ids = training(dev, dtype, num_experts=experts)
    torch.manual_seed(1)
    y = model(x, f, graph, adapters=ids)
    score(y).backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all(), name
        if "adapters" in name or name.endswith("attention.bias"):
            assert (p.grad != 0).any(), name
    assert y.dtype == dtype


def test_frozen_maps_train_their_adapters_alone(dev):
    model, x, graph, f, ids = training(dev)
    for p in model.parameters():
        p.requires_grad_(False)
    params = fe.add_adapters(model, 3, 4)
    stir(params)
    torch.manual_seed(1)
    score(model(x, f, graph, adapters=ids)).backward()
    assert all((p.grad is not None) == any(p is q for q in params) for p in model.parameters())
    full, *_ = training(dev)
    full.load_state_dict(model.state_dict())
    torch.manual_seed(1)
    score(full(x, f, graph, adapters=ids)).backward()
    want = {n: p.grad for n, p in full.named_parameters()}
    for n, p in model.named_parameters():
        if p.grad is not None:
            assert rel(p.grad, want[n]) < 1e-5, n


def test_gradients_against_differences(dev):
    """The loss along the gradient of the new parameters (0.11 a unit; it turns within steps of 0.02, so steps are
    smaller).  The results (at most 5) are off by 1e-5 of the largest, the layers' bound, so the loss, their mean with weights
    of mean size 1/2, by 2.5e-5 and a central difference over a step h by 2.5e-5 / h; of its truncation error, which goes with h^2,
    the half step's is a third of what the two differ by."""
    model, x, graph, f, ids = training(dev)
    model.eval()
    params = [p for n, p in model.named_parameters() if "adapters" in n or n.endswith("attention.bias")]

    def loss():
        return score(model(x, f, graph, adapters=ids))
    grads = torch.autograd.grad(loss(), params)
    norm = torch.sqrt(sum(t.square().sum() for t in grads)).item()
    slopes = []
    with torch.no_grad():
        for h in (0.006, 0.003):
            values = []
            for step in (h, -2 * h, h):
                for p, t in zip(params, grads):
                    p.add_(t, alpha=step / norm)
                values.append(loss().double().item())
            slopes.append((values[0] - values[1]) / (2 * h))
    print(f"gradient {norm:.4e}, differences {slopes}")
    assert abs(norm - slopes[1]) <= 2.5e-5 / 0.003 + abs(slopes[0] - slopes[1])


def test_adapter_gradients_are_those_of_the_merged_maps(dev):
    """All nodes with one adapter: the loss is that of maps W + s up down, so its gradients are s gW down^T and s up^T gW."""
    model, x, graph, f, _ = training(dev)
    model.eval()
    one = merged(model, 1)
    score(one(x, f, graph)).backward()
    score(model(x, f, graph, adapters=torch.ones(40, dtype=torch.int64, device=dev))).backward()
    checked = 0
    for (name, m), (_, o) in zip(model.named_modules(), one.named_modules()):
        if isinstance(m, fe.LinearAdapters):
            continue
        if isinstance(m, fe.EquivariantLinear):
            low = m.adapters
            gw = o.weight.grad.view(low.up.shape[1], low.up.shape[2], -1)
            # the maps before and after agree to 1e-5 of the largest in every layer; products of them to a few times that
            assert rel(low.up.grad[1], low.scale * gw @ low.down[1].transpose(1, 2)) < 1e-4, name
            assert rel(low.down.grad[1], low.scale * low.up[1].transpose(1, 2) @ gw) < 1e-4, name
            assert (low.up.grad[[0, 2]] == 0).all() and (low.down.grad[[0, 2]] == 0).all()
            checked += 1
    assert checked == 6


def test_captured_training_steps(dev):
    model, x, graph, f, ids = training(dev)
    leaves = list(model.parameters())
    plan = fe.ExpertPlan(ids, 3)
    torch.manual_seed(2)

    def step():
        loss = score(model(x, f, graph, adapters=plan))
        loss.backward()
        return loss
    g, loss = capture_step(step, leaves)
    seen = []
    for _ in range(4):
        g.replay()
        torch.cuda.synchronize()
        seen.append(loss.item())
        assert all(p.grad.isfinite().all() for p in leaves)
        model(x, f, graph, adapters=plan).sum().item()                   # the program's own work between replays
    assert len(set(seen)) == 4                                           # new masks
    model.eval()
    for p in leaves:
        p.grad = None
    g2, loss2 = capture_step(step, leaves)
    for _ in range(3):
        g2.replay()
        torch.cuda.synchronize()
        got = [p.grad.clone() for p in leaves]
        eager = torch.autograd.grad(score(model(x, f, graph, adapters=plan)), leaves)
        for a, b in zip(got, eager):
            assert rel(a, b) < 1e-5 or (b == 0).all()


def test_dropout_layer(dev):
    r = fe.Repr([0, 1, 2], 6)
    drop = fe.EquivariantDropout(r, 0.4).to(dev)
    x = torch.randn(50, 6, 9, generator=gen(40)).to(dev)
    torch.manual_seed(1)
    y = drop(x)
    torch.manual_seed(1)
    cm = drop(x.permute(2, 0, 1).contiguous(), True)
    assert torch.equal(cm.permute(1, 2, 0), y) and not torch.equal(drop(x), y)
    for a, b in ((0, 1), (1, 4), (4, 9)):                                # all of an irrep or nothing
        zero = (y[..., a:b] == 0)
        assert torch.equal(zero.all(-1), zero.any(-1))
    assert drop.eval()(x) is x and fe.EquivariantDropout(r, 0.0).train()(x) is x


def test_linear_layer_with_adapters(dev):
    for dtype, tol in ((torch.float32, 1e-5), (torch.bfloat16, 2e-2)):
        act = torch.nn.SiLU()
        for activation in (None, act):
            linear = fe.EquivariantLinear(fe.Repr([0, 1, 0], 8), fe.Repr([0, 1, 0], 12), activation=activation).to(dev)
            with torch.no_grad():
                linear.bias.copy_(torch.randn(12, 2, generator=gen(41)))
            stir(linear.add_adapters(3, 4))
            linear.to(dtype)
            f = torch.randn(4, 10, 8, 5, generator=gen(42)).to(dev, dtype)           # two leading axes
            ids = torch.randint(-1, 3, (40,), generator=gen(43)).to(dev)
            y = linear(f, fe.ExpertPlan(ids, 3))
            assert y.shape == (4, 10, 12, 5) and y.dtype == dtype
            for a in range(-1, 3):
                w = linear.weight.float()
                if a >= 0:
                    w = w + linear.adapters.scale * (linear.adapters.up[a].float() @ linear.adapters.down[a].float()).reshape(w.shape)
                alone = fe.EquivariantLinear(fe.Repr([0, 1, 0], 8), fe.Repr([0, 1, 0], 12), activation=activation).to(dev)
                with torch.no_grad():
                    alone.weight.copy_(w)
                    alone.bias.copy_(linear.bias)
                at = ids.view(4, 10) == a
                if at.any():
                    assert rel(y[at], alone(f[at].float())) < tol
            with pytest.raises(ValueError, match="a plan for 2 adapters"):
                linear(f, fe.ExpertPlan(ids, 2))


def test_refusals_of_the_dropout(dev):
    x, s = torch.randn(5, 4, 4, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            fe.feature_dropout(x, p, s)
    for seed in (s.int(), torch.zeros(2, dtype=torch.int64, device=dev), s.float()):
        with pytest.raises(ValueError, match="seed must be one int64"):
            fe.feature_dropout(x, 0.5, seed)
    with pytest.raises(fe.CUDANotAvailableError):
        fe.feature_dropout(x, 0.5, s.cpu())
    with pytest.raises(TypeError, match="float64 is not supported"):
        fe.feature_dropout(x.double(), 0.5, s)
    with pytest.raises(ValueError, match="x must be"):
        fe.feature_dropout(x, 0.5, s, [0, 1, 2])
    with pytest.raises(ValueError, match="x must be"):
        fe.feature_dropout(x, 0.5, s, [0, 1], True)
    for lv in ([], [-1]):
        with pytest.raises(ValueError, match="lvals"):
            fe.feature_dropout(x, 0.5, s, lv)
    with pytest.raises(ValueError, match="at most 32 irreps"):
        fe.feature_dropout(torch.zeros(2, 33, device=dev), 0.5, s, [0] * 33)
    with pytest.raises(NotImplementedError, match="no forward-mode"):
        with torch.autograd.forward_ad.dual_level():
            fe.feature_dropout(torch.autograd.forward_ad.make_dual(x, x), 0.5, s)


def test_refusals_of_the_attention(dev):
    src = torch.zeros(6, dtype=torch.int64, device=dev)
    graph = fe.Graph(src, src, 3)
    qk, ls = torch.randn(3, 8, 4, device=dev), torch.zeros((), device=dev)
    bias, b = torch.zeros(5, 2, device=dev), torch.zeros(6, dtype=torch.int32, device=dev)
    call = lambda qk=qk, heads=2, ls=ls, **kw: fe.edge_attention_weights(qk, graph, heads, ls, **kw)
    for bad in (qk[:, :7], torch.randn(3, 8, device=dev), torch.randn(3, 0, 4, device=dev), qk[:, :6]):
        with pytest.raises(ValueError, match="qk must be"):
            call(bad)
    with pytest.raises(ValueError, match="rows but the graph has 3"):
        call(qk[:2])
    for heads in (0, 1025):
        with pytest.raises(ValueError, match="num_heads must be"):
            call(heads=heads)
    with pytest.raises(ValueError, match="heads dividing mult"):
        call(heads=3)
    with pytest.raises(ValueError, match="log_scale must be one number"):
        call(ls=torch.zeros(2, device=dev))
    with pytest.raises(TypeError, match="float64"):
        call(qk.double())
    for kw in (dict(bias=bias), dict(buckets=b)):
        with pytest.raises(ValueError, match="come together"):
            call(**kw)
    for bad in (bias[:, :1], bias[0], torch.zeros(0, 2, device=dev), torch.zeros(4097, 2, device=dev)):
        with pytest.raises(ValueError, match="bias must be"):
            call(bias=bad, buckets=b)
    with pytest.raises(ValueError, match="buckets must be"):
        call(bias=bias, buckets=b[:5])
    with pytest.raises(TypeError, match="int32 or int64"):
        call(bias=bias, buckets=b.float())
    with pytest.raises(fe.CUDANotAvailableError):
        call(bias=bias, buckets=b.cpu())
    with pytest.raises(ValueError, match="needs a seed"):
        call(dropout=0.5)
    with pytest.raises(ValueError, match="between 0 and 1"):
        call(dropout=1.5)
    with pytest.raises(ValueError, match="needs distances"):
        call(decay=1.0)
    with pytest.raises(ValueError, match="must not be negative"):
        call(decay=-1.0)
    with pytest.raises(ValueError, match="distances must be"):
        call(decay=1.0, distances=torch.rand(5, device=dev))
    Q = torch.randn(6, 2, 4, device=dev)
    for q, k in ((Q, Q[:, :1]), (Q[:5], Q[:5]), (Q[0], Q[0])):
        with pytest.raises(ValueError):
            fe.edge_attention_weights_qk(q, k, graph, ls)
    with pytest.raises(TypeError, match="different dtypes"):
        fe.edge_attention_weights_qk(Q, Q.half(), graph, ls)
    with pytest.raises(ValueError, match="needs the edges' buckets"):
        fe.EquivariantEdgeAttention(2, 4, bias_buckets=5).to(dev).attention_weights(Q, Q, graph)
    with pytest.raises(TypeError, match="must be float32"):
        fe.distance_buckets(torch.rand(3, device=dev).double(), torch.rand(2, device=dev))
    with pytest.raises(ValueError, match="expected"):
        fe.distance_buckets(torch.rand(3, 1, device=dev), torch.rand(2, device=dev))


def test_refusals_of_the_adapters(dev):
    plan = fe.ExpertPlan(torch.zeros(6, dtype=torch.int64, device=dev), 3)
    x, w = torch.randn(4, 6, 8, device=dev), torch.randn(2, 5, 8, device=dev)
    d, u, b = torch.randn(3, 2, 4, 8, device=dev), torch.randn(3, 2, 5, 4, device=dev), torch.randn(5, 1, device=dev)
    call = lambda x=x, w=w, d=d, u=u, plan=plan, lv=(0, 1), b=b, s=1.0: fe.adapter_linear(x, w, d, u, plan, lv, b, s)
    call()
    for bad in (x[:3], x[:, :5], x[..., :7], x[0]):
        with pytest.raises(ValueError, match="x must be"):
            call(x=bad)
    for bad in (w[:1], w[:, :4], w.view(10, 8)[:9], w[0, 0]):
        with pytest.raises(ValueError, match="weight must be"):
            call(w=bad)
    for bad in (d[:2], d[:, :1], d[0], d[:, :, :0], torch.randn(3, 2, 65, 8, device=dev)):
        with pytest.raises(ValueError, match="down must be"):
            call(d=bad)
    for bad in (u[:2], u[:, :1], u[..., :3], u[0]):
        with pytest.raises(ValueError, match="up must be"):
            call(u=bad)
    for bad in (b[:4], b[:, 0], torch.randn(5, 2, device=dev)):
        with pytest.raises(ValueError, match="bias must be"):
            call(b=bad)
    for kw in (dict(w=w.half()), dict(d=d.half()), dict(u=u.half()), dict(b=b.half())):
        with pytest.raises(TypeError, match="different dtypes"):
            call(**kw)
    with pytest.raises(TypeError, match="float64"):
        call(x=x.double())
    with pytest.raises(ValueError, match="scale must be finite"):
        call(s=float("nan"))
    with pytest.raises(ValueError, match="one adapter"):
        call(plan=fe.ExpertPlan(torch.zeros(3, 2, dtype=torch.int64, device=dev), 3))
    with pytest.raises(ValueError, match="lvals"):
        call(lv=())
    with pytest.raises(fe.CUDANotAvailableError):
        call(w=w.cpu())


def test_a_decay_that_is_zero_in_float32_is_refused(dev):
    src = torch.zeros(6, dtype=torch.int64, device=dev)
    graph, qk = fe.Graph(src, src, 3), torch.randn(3, 8, 4, device=dev)
    with pytest.raises(ValueError, match="is 0 in float32"):
        fe.edge_attention_weights(qk, graph, 2, torch.zeros((), device=dev), decay=1e-60, distances=torch.rand(6, device=dev))
