"""Layer norm kernels (csrc/layernorm.hip) against the float64 oracle on the same inputs.

Bounds, with u = 2^-24 (float32), h(t) half a step of the stored type t (2^-24, 2^-11, 2^-8 relative)
and K = 64: a lane adds at most 32 values in a row and 8 more levels join lanes and waves (the kernels
for very wide rows add width / 1024 values a thread), so a sum is off by at most K u of its absolute
terms, and with it the mean by K u max|x| and xh by u K A, A = |xh| + max|x| rstd.  The other terms
follow from the formulas term by term."""
import pytest
import torch

import flash_eq as fe
from flash_eq import ops
from oracle import experts as OE

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}     # half a subnormal step
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# one element; no spread; odd; each lane-group form; a workgroup a row; rows beyond its registers, odd too
SIZES = [(1, 1), (3, 2), (5, 7), (100, 192), (33, 55), (7, 1000), (64, 1024), (17, 1152), (9, 4096), (3, 8192),
         (2, 8200), (2, 20000), (3, 16391), (2050, 64), (5000, 8), (300, 896), (4, 2049),
         # a last vector that shares elements, in each form
         (6, 9), (40, 63), (21, 257), (8, 515), (5, 1027), (3, 6978), (3, 8191), (70, 8193)]


def within(got, want, tol, dtype):
    err = (got.detach().double().cpu() - want).abs()
    bad = err > tol + TINY[dtype]
    assert not bad.any(), (float((err - tol).max()), int(bad.sum()), got.shape)


def check(dev, x, w, b, gy, eps=1e-5):
    xd = x.detach().double().cpu().requires_grad_()
    wd = w.double().cpu().requires_grad_() if w is not None else None
    bd = b.double().cpu().requires_grad_() if b is not None else None
    yr = OE.layer_norm(xd, wd, bd, eps)
    leaves = [t for t in (xd, wd, bd) if t is not None]
    grads = dict(zip("xwb", torch.autograd.grad(yr, leaves, gy.double().cpu()))) if w is not None else \
        {"x": torch.autograd.grad(yr, [xd], gy.double().cpu())[0]}

    xl = x.detach().requires_grad_()
    wl, bl = (t.clone().requires_grad_() if t is not None else None for t in (w, b))
    y = ops.layer_norm(xl, wl, bl, eps)
    outs = torch.autograd.grad(y, [t for t in (xl, wl, bl) if t is not None], gy)

    x0, g0 = xd.detach(), gy.double().cpu()
    width = x0.shape[-1]
    K = 64 + width / 1024
    mu = x0.mean(-1, keepdim=True)
    rs = 1 / torch.sqrt(((x0 - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = ((x0 - mu) * rs).abs()
    A = xh + x0.abs().amax(-1, keepdim=True) * rs
    wa = wd.detach().abs() if wd is not None else 1.0
    ba = bd.detach().abs() if bd is not None else 0.0
    # the variance's relative error (2 K u A per term) scales xh once more
    tol_y = HALF[x.dtype] * yr.detach().abs() + U * K * (A * wa + xh * (A * A).mean(-1, keepdim=True) * wa + ba)
    within(y, yr.detach(), tol_y, x.dtype)
    assert torch.equal(ops.layer_norm(x.detach(), w, b, eps), y.detach())       # the form without gradients
    h = (g0 * wa).abs()
    E = 1 + (A * A).mean(-1, keepdim=True)
    tol_x = HALF[x.dtype] * grads["x"].abs() + U * K * rs * E * (
        h + h.mean(-1, keepdim=True) + A * (h * A).mean(-1, keepdim=True))
    within(outs[0], grads["x"], tol_x, x.dtype)
    if w is not None:
        # a lane's run over rows adds at most rows / 16 values (16 rows a workgroup at least share the sums)
        Kr = K + 64 + x0.numel() / width / 16
        dims = tuple(range(x0.dim() - 1))
        tol_w = HALF[w.dtype] * grads["w"].abs() + U * Kr * (g0.abs() * A * E).sum(dims)
        within(outs[1], grads["w"], tol_w, w.dtype)
        within(outs[2], grads["b"], HALF[w.dtype] * grads["b"].abs() + U * Kr * g0.abs().sum(dims), w.dtype)


def inputs(dev, rows, width, dtype, seed, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, width, generator=g) + shift).to(dev, dtype)
    w = (1 + 0.3 * torch.randn(width, generator=g)).to(dev, dtype)
    b = (0.3 * torch.randn(width, generator=g)).to(dev, dtype)
    gy = torch.randn(rows, width, generator=g).to(dev, dtype)
    return x, w, b, gy


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", SIZES)
def test_sizes(dev, rows, width, dtype):
    check(dev, *inputs(dev, rows, width, dtype, rows + width))


def test_a_large_mean_and_a_large_epsilon(dev):
    x, w, b, gy = inputs(dev, 40, 320, torch.float32, 1, shift=1000.0)
    check(dev, x, w, b, gy)
    check(dev, x, w, b, gy, eps=3.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_parameters_and_with_parameters_of_another_type(dev, dtype):
    x, w, b, gy = inputs(dev, 37, 96, dtype, 2)
    check(dev, x, None, None, gy)
    other = torch.float32 if dtype != torch.float32 else torch.bfloat16
    check(dev, x, w.to(other), b.to(other), gy)


def test_only_the_gradients_that_are_wanted(dev):
    x, w, b, gy = inputs(dev, 50, 130, torch.float32, 3)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    every = torch.autograd.grad(ops.layer_norm(*leaves), leaves, gy)
    for i in range(3):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        (one,) = torch.autograd.grad(ops.layer_norm(*args), [args[i]], gy)
        assert torch.equal(one, every[i])
    w1 = w.clone().requires_grad_()             # a weight without a bias
    (gw,) = torch.autograd.grad(ops.layer_norm(x, w1), [w1], gy)
    assert torch.equal(gw, every[1])
    b1 = b.clone().requires_grad_()             # a bias without a weight
    (gb,) = torch.autograd.grad(ops.layer_norm(x, None, b1), [b1], gy)
    assert torch.equal(gb, every[2])


@pytest.mark.parametrize("width,cut", [(64, (8, 72)), (64, (3, 67)), (33, (1, 34))])
def test_rows_of_a_wider_table_and_strided_gradients(dev, width, cut):
    """A column slice is read in place: rows apart, 16-byte aligned or not."""
    g = torch.Generator().manual_seed(4)
    table = torch.randn(45, 80, generator=g).to(dev)
    x = table[:, cut[0]:cut[1]]
    assert not x.is_contiguous() and x.shape[1] == width
    _, w, b, _ = inputs(dev, 1, width, torch.float32, 5)
    gy = torch.randn(45, 80, generator=g).to(dev)[:, cut[0]:cut[1]]
    check(dev, x, w, b, gy)
    a = ops.layer_norm(x, w, b)
    assert a.is_contiguous()
    assert torch.equal(a, ops.layer_norm(x.contiguous(), w, b))


def test_shapes_and_broadcast_gradients(dev):
    x, w, b, _ = inputs(dev, 24, 40, torch.float32, 6)
    x4 = x.view(2, 3, 4, 40)
    assert torch.equal(ops.layer_norm(x4, w, b), ops.layer_norm(x, w, b).view(2, 3, 4, 40))
    t = x4.transpose(0, 2)                      # rows in another order
    assert torch.equal(ops.layer_norm(t, w, b), ops.layer_norm(t.contiguous(), w, b))
    v = x[0]
    assert torch.equal(ops.layer_norm(v, w, b), ops.layer_norm(x, w, b)[0])
    xl = x.clone().requires_grad_()
    (ops.layer_norm(xl, w, b) * 2).sum().backward()         # the gradient of a sum has stride 0
    gy = torch.full_like(x, 2.0)
    xm = x.clone().requires_grad_()
    ops.layer_norm(xm, w, b).backward(gy)
    assert torch.equal(xl.grad, xm.grad)


def test_no_rows(dev):
    w = torch.ones(12, device=dev, requires_grad=True)
    b = torch.zeros(12, device=dev, requires_grad=True)
    x = torch.empty(0, 12, device=dev, requires_grad=True)
    y = ops.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty(0, 12, device=dev))
    assert y.shape == gx.shape == (0, 12)
    assert not gw.any() and not gb.any()


@pytest.mark.parametrize("rows,width", [(70, 192), (5, 1500), (3, 9001)])
def test_infinities_and_nan_stay_in_their_rows(dev, rows, width):
    x, w, b, gy = inputs(dev, rows, width, torch.float32, 7)
    xl = x.clone().requires_grad_()
    y = ops.layer_norm(xl, w, b)
    (gx,) = torch.autograd.grad(y, [xl], gy)
    x2 = x.clone()
    x2[0, 1], x2[2, 3] = float("inf"), float("nan")
    x2.requires_grad_()
    y2 = ops.layer_norm(x2, w, b)
    (gx2,) = torch.autograd.grad(y2, [x2], gy)
    assert torch.isnan(y2[0]).any() and torch.isnan(y2[2]).all()
    keep = [r for r in range(rows) if r not in (0, 2)]
    assert torch.equal(y2[keep], y[keep]) and torch.equal(gx2[keep], gx[keep])


@pytest.mark.parametrize("width", [192, 1500])
def test_the_same_bits_on_every_run(dev, width):
    x, w, b, gy = inputs(dev, 9000, width, torch.float32, 8)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(ops.layer_norm(*leaves), leaves, gy)
    for _ in range(3):
        again = torch.autograd.grad(ops.layer_norm(*leaves), leaves, gy)
        assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_captured_step_and_another_stream(dev):
    from flash_eq.capture import capture_step
    x, w, b, gy = inputs(dev, 600, 192, torch.float32, 9)
    norm = fe.InvariantLayerNorm(192).to(dev)
    x.requires_grad_()

    def step():
        loss = (norm(x) * gy).sum(-1).mean()
        loss.backward()
        return loss

    graph, loss = capture_step(step, [x, *norm.parameters()])
    for k in range(4):
        with torch.no_grad():
            x.copy_(inputs(dev, 600, 192, torch.float32, 20 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.grad.clone() for t in (x, norm.weight, norm.bias)]
        y = ops.layer_norm(x, norm.weight, norm.bias)
        want = torch.autograd.grad((y * gy).sum(-1).mean(), [x, norm.weight, norm.bias])
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2 = ops.layer_norm(x, norm.weight, norm.bias)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y2, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [5, 17, 100, 1030, 8200])
def test_unaligned_tables(dev, width, dtype):
    """Tables and parameters from an address that is a multiple of their element alone: the bits of aligned ones."""
    x, w, b, gy = inputs(dev, 23, width, dtype, width)

    def apart(t):
        return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    def step(x, w, b, gy):
        x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
        y = ops.layer_norm(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, [x, w, b], gy))

    for one, two in zip(step(x, w, b, gy), step(*(apart(t) for t in (x, w, b, gy)))):
        assert torch.equal(one, two)


def test_past_32_bit_offsets(dev):
    """Rows whose elements lie behind the first 2^31, read and written at their places."""
    rows, width = 2 ** 21 + 3, 1030              # 2.2e9 elements
    x = torch.empty(rows, width, device=dev, dtype=torch.bfloat16)
    x[-4:] = torch.randn(4, width, generator=torch.Generator().manual_seed(1)).to(dev, torch.bfloat16)
    x[:-4] = 0
    x.requires_grad_()
    y = ops.layer_norm(x)
    y0 = ops.layer_norm(x.detach()[-4:].clone().requires_grad_())
    assert torch.equal(y[-4:], y0) and not y[:4].any() and not y[rows // 2].any()
    gy = torch.zeros_like(x)
    gy[-4:] = 1.0
    (gx,) = torch.autograd.grad(y, [x], gy)
    x0 = x.detach()[-4:].clone().requires_grad_()
    (g0,) = torch.autograd.grad(ops.layer_norm(x0), [x0], gy[-4:].clone())
    assert torch.equal(gx[-4:], g0) and not gx[:4].any()


def test_inputs_changed_before_the_backward_are_refused(dev):
    x, w, b, gy = inputs(dev, 8, 40, torch.float32, 12)
    for i in range(2):
        args = [x.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()]
        y = ops.layer_norm(*args)
        with torch.no_grad():
            args[i].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward(gy)


def test_no_forward_mode(dev):
    x = torch.randn(4, 8, device=dev)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            ops.layer_norm(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


def test_refusals(dev):
    x = torch.randn(4, 8, device=dev)
    with pytest.raises(RuntimeError, match="exceeds 2\\^24"):
        ops.layer_norm(torch.zeros(1, 2 ** 24 + 1, device=dev))
    with pytest.raises(TypeError, match="float64"):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError, match=r"weight must have shape \(8,\)"):
        ops.layer_norm(x, torch.ones(7, device=dev))
    with pytest.raises(TypeError, match="different dtypes"):
        ops.layer_norm(x, torch.ones(8, device=dev), torch.ones(8, device=dev, dtype=torch.float16))
    with pytest.raises(fe.CUDANotAvailableError):
        ops.layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="last axis"):
        ops.layer_norm(torch.empty(3, 0, device=dev))
    xl = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(ops.layer_norm(xl).pow(2).sum(), [xl], create_graph=True)
    with pytest.raises(RuntimeError):           # no second derivative, and not a wrong one
        gx.sum().backward()
    # float64 modules take PyTorch's layer norm, as the other norms do
    norm = fe.InvariantLayerNorm(8).to(dev).double()
    assert torch.equal(norm(x.double()), torch.nn.functional.layer_norm(x.double(), (8,), norm.weight, norm.bias, 1e-5))


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_the_rows_alone(dev, dtype):
    """Frozen or absent parameters: the bits of the call that has their gradients too, in each form of few rows."""
    for rows, width in ((1, 5), (8, 3000), (7, 8192), (128, 192), (20, 1000), (256, 40), (3, 9000), (40, 9001)):
        g = torch.Generator().manual_seed(rows)
        x, gy = (torch.randn(rows, width, generator=g).to(dev, dtype) for _ in range(2))
        w, b = (torch.randn(width, generator=g).to(dev, dtype).requires_grad_() for _ in range(2))
        x.requires_grad_()
        y = ops.layer_norm(x, w, b)
        both = torch.autograd.grad(y, [x, w, b], gy, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(y, [x], gy)[0], both)
        frozen = ops.layer_norm(x, w.detach(), b.detach())
        assert torch.equal(torch.autograd.grad(frozen, [x], gy)[0], both)
        ones = torch.ones(width, device=dev, dtype=dtype, requires_grad=True)
        plain = torch.autograd.grad(ops.layer_norm(x, ones), [x, ones], gy)[0]
        assert torch.equal(torch.autograd.grad(ops.layer_norm(x), [x], gy)[0], plain)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_widest_rows(dev, dtype):
    x, w, b, gy = inputs(dev, 3, 2 ** 24, dtype, 40)
    check(dev, x, w, b, gy)
