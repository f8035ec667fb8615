"""Long sums of the biased edge attention's gradients."""
import pytest
import torch

import flash_eq as fe

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("heads,buckets,log_edges", [(1024, 4096, 20), (1, 4096, 22), (8, 100, 20)])
def test_bias_gradient_of_many_edges_in_one_bucket(dev, heads, buckets, log_edges):
    """Two edges into every node, one in bucket 0 and one in the last; all logits 0, so both weights are 1/2, and of the gradients
    g of the first and 0 of the second the logits' are g / 4 and -g / 4: all of them exact in float32.  What is off is the sums of
    equal numbers, whose roundings do not cancel.  A table in LDS takes 2048 edges a slot before it is added to its workgroup's
    partial; 512 workgroups at most share the edges."""
    E = 1 << log_edges
    n = E // 2
    dst = torch.arange(n, device=dev).repeat_interleave(2)
    graph = fe.Graph(torch.zeros_like(dst), dst, n)
    bucket = (torch.arange(E, device=dev) % 2 * (buckets - 1)).int()
    g = (1 + torch.rand(heads, generator=torch.Generator().manual_seed(1))).to(dev)
    bias = torch.zeros(buckets, heads, device=dev, requires_grad=True)
    qk = torch.zeros(n, 2 * heads, 1, device=dev)
    w = fe.edge_attention_weights(qk, graph, heads, torch.zeros((), device=dev), bias=bias, buckets=bucket)
    assert (w[:2] == 0.5).all() and (w[-2:] == 0.5).all()
    gw = torch.zeros(n, 2, heads, device=dev)
    gw[:, 0] = g
    (gb,) = torch.autograd.grad(w, bias, gw.view(E, heads))
    want = n * (g.double() / 4)
    # 2048 additions of a slot, 256 tables, the partial's additions (each of 2048 edges and more) and the result's rounding
    tol = (2048 + 256 + E / 8 / 2048 + 1) * U * want
    for got, sign in ((gb[0], 1), (gb[-1], -1)):
        err = (got.double() - sign * want).abs()
        assert (err <= tol).all(), (err / want / U).max().item()
    assert not gb[1:-1].any()
    del qk, w, gw, gb
    torch.cuda.empty_cache()
