"""The float64 oracle of the fine-tuning operators: known answers, closed forms, differences."""
import math

import pytest
import torch

from oracle import finetune as OF


def gen(seed):
    return torch.Generator().manual_seed(seed)


def test_generator_known_answers():
    """The known answers that the generator's authors publish for Philox 4 x 32 with ten rounds."""
    ones = 0xFFFFFFFF
    assert OF.philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert OF.philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert OF.philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_factors():
    f = OF.factors(0, 16, 0.5)
    words = [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert f[:8].tolist() == [2.0 * (v >= 32768) for w in words for v in (w & 0xFFFF, w >> 16)]
    assert OF.factors(-1, 3, 0.3).tolist() == OF.factors(2 ** 64 - 1, 3, 0.3).tolist()
    assert OF.factors(5, 100, 0.0).eq(1).all() and OF.factors(5, 100, 1.0).eq(0).all()
    f = OF.factors(7, 40000, 0.1)                       # a binomial share: 5 standard deviations
    limit = round(6553.6)
    assert abs((f == 0).double().mean() - limit / 65536) < 5 * math.sqrt(0.09 / 40000)
    assert f.max() == 65536 / (65536 - limit)


def test_dropout_layouts():
    x = torch.randn(5, 3, 9, generator=gen(0), dtype=torch.float64)
    x[0, 0, 0] = float("nan")
    y = OF.dropout(x, 0.5, 11, [0, 1, 2])
    cm = OF.dropout(x.permute(2, 0, 1).contiguous(), 0.5, 11, [0, 1, 2], True)
    assert torch.equal(cm.nan_to_num(nan=7.0), y.permute(2, 0, 1).nan_to_num(nan=7.0))
    f = OF.factors(11, 5 * 3 * 3, 0.5).view(5, 3, 3)
    for i in range(5):
        for c in range(3):
            for r, (a, b) in enumerate(((0, 1), (1, 4), (4, 9))):
                want = torch.zeros(b - a, dtype=torch.float64) if f[i, c, r] == 0 else x[i, c, a:b] * 2
                assert torch.equal(y[i, c, a:b].nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


def graph(seed, nodes=6, edges=40):
    g = gen(seed)
    return torch.randint(0, nodes, (edges,), generator=g), torch.randint(0, nodes - 1, (edges,), generator=g)


def test_attention_is_softmax_of_the_biased_logits():
    src, dst = graph(1)
    g = gen(2)
    qk = torch.randn(6, 8, 4, generator=g, dtype=torch.float64)
    bias, bucket = torch.randn(5, 2, generator=g, dtype=torch.float64), torch.randint(0, 5, (40,), generator=g)
    q, k = OF.node_qk(qk, 2, src, dst)
    w = OF.edge_attention(q, k, dst, 6, torch.tensor(-0.7, dtype=torch.float64), None, 0.0, bias, bucket)
    for e in range(40):
        for h in range(2):
            z = [math.exp(-0.7) * (qk[dst[f], 2 * h:2 * h + 2].reshape(-1) @ qk[src[f], 4 + 2 * h:6 + 2 * h].reshape(-1))
                 + bias[bucket[f], h] for f in range(40) if dst[f] == dst[e]]
            m = max(z)
            own = math.exp(-0.7) * (q[e, h] @ k[e, h]) + bias[bucket[e], h]
            assert abs(w[e, h] - math.exp(own - m) / (sum(math.exp(v - m) for v in z) + 1e-8)) < 1e-13


def test_attention_gradients_by_differences_and_forbidden_buckets():
    src, dst = graph(3, 5, 14)
    g = gen(4)
    qk = torch.randn(5, 4, 3, generator=g, dtype=torch.float64, requires_grad=True)
    bias = torch.randn(4, 2, generator=g, dtype=torch.float64)
    bias[3] = float("-inf")
    bias[1, 0] = float("-inf")
    bias.requires_grad_()
    bucket = torch.randint(0, 5, (14,), generator=g)                # 4: outside, no bias
    ls = torch.tensor(0.3, dtype=torch.float64, requires_grad=True)
    dist = torch.rand(14, generator=g, dtype=torch.float64, requires_grad=True)

    def f(qk, finite, ls, dist):
        b = torch.where(bias.detach() == float("-inf"), bias.detach(), finite)
        q, k = OF.node_qk(qk, 2, src, dst)
        return OF.edge_attention(q, k, dst, 5, ls, dist, 2.0, b, bucket, 0.25, 9)

    finite = bias.detach().clamp(min=-9).requires_grad_()
    assert torch.autograd.gradcheck(f, (qk, finite, ls, dist), eps=1e-6, atol=1e-6)
    w = f(qk, finite, ls, dist)
    assert (w[bucket == 3] == 0).all() and (w[bucket == 1][:, 0] == 0).all()
    none = OF.edge_attention(*OF.node_qk(qk, 2, src, dst), dst, 5, ls, None, 0.0, torch.full((1, 2), float("-inf"), dtype=torch.float64),
                             torch.zeros(14, dtype=torch.int64))
    assert (none == 0).all()


def test_log_scale_gradient_is_the_queries_dot_their_gradient():
    src, dst = graph(5)
    qk = torch.randn(6, 8, 4, generator=gen(6), dtype=torch.float64, requires_grad=True)
    ls = torch.tensor(0.1, dtype=torch.float64, requires_grad=True)
    w = OF.edge_attention(*OF.node_qk(qk, 2, src, dst), dst, 6, ls)
    gqk, gls = torch.autograd.grad(w, [qk, ls], torch.randn(40, 2, generator=gen(7), dtype=torch.float64))
    assert abs((qk[:, :4] * gqk[:, :4]).sum() - gls) < 1e-12
    assert abs((qk[:, 4:] * gqk[:, 4:]).sum() - gls) < 1e-12


def test_adapter_rows_are_a_merged_map():
    g = gen(8)
    lv = [0, 1, 0]
    x = torch.randn(5, 7, 4, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(3, 6, 4, generator=g, dtype=torch.float64, requires_grad=True)
    down = torch.randn(2, 3, 2, 4, generator=g, dtype=torch.float64, requires_grad=True)
    up = torch.randn(2, 3, 6, 2, generator=g, dtype=torch.float64, requires_grad=True)
    bias = torch.randn(6, 2, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([1, 0, -1, 1, 5, 0, 1])
    y = OF.adapter_linear(x, w, down, up, ids, lv, bias, 0.5)
    rep = [0, 1, 1, 1, 2]
    for i, a in enumerate(ids.tolist()):
        for d, r in enumerate(rep):
            m = w[r] + (0.5 * up[a, r] @ down[a, r] if a in (0, 1) else 0)
            want = m @ x[d, i] + (bias[:, 0] if d == 0 else bias[:, 1] if d == 4 else 0)
            assert (y[d, i] - want).abs().max() < 1e-13
    assert torch.autograd.gradcheck(lambda *t: OF.adapter_linear(t[0], t[1], t[2], t[3], ids, lv, t[4], 0.5), (x, w, down, up, bias))


def test_buckets():
    b = OF.buckets(torch.tensor([0.0, 1.0, 0.99, 2.5, float("nan"), -1.0]), torch.tensor([1.0, 2.0]))
    assert b.tolist() == [0, 1, 0, 2, 0, 0]
