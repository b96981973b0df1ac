"""GPU: LayerNorm of 16- and 32-bit tensors (coat_amd.activation.norm) against its definition in 64 bits.

Bounds.  u = half a step of the output's type.  fp32 sums add at most 8 values per 2048 columns (or 32 in registers) one after the
other and then 22 partial sums: K = 64 + N / 256 roundings of 2^-24 cover a sum and the few operations around it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(dev, M, N, dtype, wdtype, seed, shift=0.3, sliced=False):
    g = torch.Generator().manual_seed(seed)

    def rows(t):
        t = t.to(dtype)
        if not sliced:
            return t.to(dev)
        wide = torch.full((M, N + 11), float("nan"), dtype=dtype)  # what lies beside the slice must not be read into a sum
        wide[:, 3:3 + N] = t
        return wide.to(dev)[:, 3:3 + N]

    x = rows(torch.randn(M, N, generator=g) * (0.5 + torch.rand(M, 1, generator=g)) + shift)
    dy = rows(torch.randn(M, N, generator=g) * 0.1)
    w = None if wdtype is None else (1 + 0.2 * torch.randn(N, generator=g)).to(wdtype).to(dev)
    b = None if wdtype is None else (0.1 * torch.randn(N, generator=g)).to(wdtype).to(dev)
    return x, dy, w, b


def check_forward(x, w, b, eps, got):
    y, mean, rstd = got
    N = x.shape[-1]
    K = (64 + N / 256) * 2.0 ** -24
    xd = x.double()
    m = xd.mean(-1)
    r = ((xd - m[..., None]).square().mean(-1) + eps).rsqrt()
    h = (xd - m[..., None]) * r[..., None]
    wd = torch.ones(N, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    want = h * wd + bd
    top = xd.abs().amax(-1)
    assert y.dtype == x.dtype and y.shape == x.shape and mean.shape == rstd.shape == x.shape[:-1]
    assert ((mean.double() - m).abs() <= K * top).all()
    # the variance is off by K of itself and by the square of what the mean is off
    assert ((rstd.double() - r).abs() <= r * (K + (K * top * r) ** 2)).all()
    bound = half_step(x.dtype) * want.abs() + K * (2 * (top * r)[..., None] * wd.abs() + want.abs() + bd.abs()) + torch.finfo(x.dtype).tiny
    assert ((y.double() - want).abs() <= bound).all(), ((y.double() - want).abs() / bound).max()


def check_backward(dy, x, mean, rstd, w, got):
    dx, dw, db = got
    N, M = x.shape[-1], x.numel() // x.shape[-1]
    K, Kr = (64 + N / 256) * 2.0 ** -24, (64 + M / 32) * 2.0 ** -24  # at most M / 32 rows one after the other in a partial row
    xd, g, m, r = (t.double().reshape(M, -1) for t in (x, dy, mean, rstd))
    wd = torch.ones(N, dtype=torch.float64, device=x.device) if w is None else w.double()
    h, hb, t = (xd - m) * r, (xd.abs() + m.abs()) * r, g * wd
    want = r * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
    if dx is not None:
        err = (dx.double().reshape(M, N) - want).abs()
        size = r * (t.abs() + t.abs().mean(1, keepdim=True) + 2 * hb * (t.abs() * hb).mean(1, keepdim=True))
        bound = half_step(x.dtype) * want.abs() + K * size + torch.finfo(x.dtype).tiny
        assert dx.shape == x.shape and dx.dtype == x.dtype
        assert (err <= bound).all(), (err / bound).max()
    for name, grad, value, size in (("dw", dw, (g * h).sum(0), (g.abs() * hb).sum(0)), ("db", db, g.sum(0), g.abs().sum(0))):
        if grad is not None:
            err = (grad.double() - value).abs()
            bound = half_step(w.dtype) * value.abs() + (Kr + 4 * 2.0 ** -24) * size + torch.finfo(w.dtype).tiny
            assert grad.shape == (N,) and grad.dtype == w.dtype
            assert (err <= bound).all(), (name, (err / bound).max())


SHAPES = [(1, 1), (3, 1), (5, 7), (1, 64), (70, 65), (33, 128), (9, 200), (17, 512), (130, 1000), (4, 1024), (3, 1025), (40, 2048),
          (11, 2049), (5, 4096), (257, 4099), (6, 8192), (3, 8200), (2, 16384), (3, 16385), (2, 40001), (3000, 33), (2100, 1024)]


@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32"), ("bf16", None), ("fp32", "fp16")])
def test_forward_and_backward(dev, M, N, dtype, wdtype):
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    wd = None if wdtype is None else TYPES[wdtype]
    x, dy, w, b = make(dev, M, N, TYPES[dtype], wd, M * 31 + N)
    out = layer_norm_forward(x, w, b, 1e-5)
    check_forward(x, w, b, 1e-5, out)
    grads = layer_norm_backward(dy, x, out[1], out[2], w)
    check_backward(dy, x, out[1], out[2], w, grads)
    assert (grads[1] is None) == (w is None) == (grads[2] is None)


@pytest.mark.parametrize("M,N", [(5, 7), (70, 65), (130, 1000), (11, 2049), (257, 4099), (3, 16385), (50, 4096)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_column_slices_of_wider_tensors(dev, M, N, dtype):
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    x, dy, w, b = make(dev, M, N, TYPES[dtype], torch.float32, 5, sliced=True)
    assert not x.is_contiguous() or M == 1
    out = layer_norm_forward(x, w, b, 1e-5)
    check_forward(x, w, b, 1e-5, out)
    check_backward(dy, x, out[1], out[2], w, layer_norm_backward(dy, x, out[1], out[2], w))


def test_other_strides_give_the_same_bits(dev):
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    x, dy, w, b = make(dev, 60, 96, torch.bfloat16, torch.bfloat16, 3)
    want = layer_norm_forward(x, w, b)
    grads = layer_norm_backward(dy, x, want[1], want[2], w)
    x3 = x.view(5, 12, 96)
    forms = [x3, x3.transpose(0, 1).contiguous().transpose(0, 1), x.t().contiguous().t().view(5, 12, 96)]
    for form in forms:
        y, mean, rstd = layer_norm_forward(form, w, b)
        assert y.shape == (5, 12, 96) and mean.shape == (5, 12)
        assert torch.equal(y.view(60, 96), want[0]) and torch.equal(mean.view(-1), want[1]) and torch.equal(rstd.view(-1), want[2])
        for a, e in zip(layer_norm_backward(dy.view(5, 12, 96), form, mean, rstd, w), grads):
            assert torch.equal(a.reshape(e.shape), e)
    w2 = torch.stack((w, w), 1)[:, 0]  # a strided weight
    assert torch.equal(layer_norm_forward(x, w2, b)[0], want[0])
    one = x[:1].expand(60, 96)  # one row repeated, dy a scalar's expansion
    y, mean, rstd = layer_norm_forward(one, w, b)
    assert torch.equal(y, want[0][:1].expand(60, 96))
    ones = torch.ones((), dtype=x.dtype, device=dev).expand(60, 96)
    check_backward(ones, one, mean, rstd, w, layer_norm_backward(ones, one, mean, rstd, w))


def test_no_rows_and_parts_of_the_gradients(dev):
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    w = torch.ones(40, device=dev)
    x = torch.empty(0, 3, 40, device=dev)
    y, mean, rstd = layer_norm_forward(x, w, w)
    assert y.shape == x.shape and mean.shape == (0, 3)
    dx, dw, db = layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(w))
    x, dy, w, b = make(dev, 300, 1000, torch.bfloat16, torch.float32, 9)
    _, mean, rstd = layer_norm_forward(x, w, b)
    full = layer_norm_backward(dy, x, mean, rstd, w)
    for keep in range(1, 8):
        kw = dict(x_grad=bool(keep & 1), weight_grad=bool(keep & 2), bias_grad=bool(keep & 4))
        for k, (a, e) in enumerate(zip(layer_norm_backward(dy, x, mean, rstd, w, **kw), full)):
            assert (a is None) if not keep >> k & 1 else torch.equal(a, e), (keep, k)


def test_rows_far_from_zero_constant_rows_and_values_that_are_not_finite(dev):
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    for N in (100, 1000, 5000, 20000):
        x, dy, w, b = make(dev, 20, N, torch.float32, torch.float32, 1, shift=1000.0)  # the two-pass variance keeps its digits
        check_forward(x, w, b, 1e-5, layer_norm_forward(x, w, b, 1e-5))
        const = torch.full((3, N), 2.5, device=dev)
        y, mean, rstd = layer_norm_forward(const, w, b, 1e-5)
        assert torch.equal(mean, const[:, 0]) and torch.equal(y, b.expand(3, N))
        assert torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5), rtol=1e-6)
        x[7, N // 2], x[9, 0] = float("nan"), float("inf")
        y, mean, rstd = layer_norm_forward(x, w, b)
        bad = torch.zeros(20, dtype=torch.bool, device=dev)
        bad[7] = bad[9] = True
        assert torch.equal(torch.isnan(y).any(1), bad) and torch.isfinite(y[~bad]).all()
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w)
        assert torch.isfinite(dx[~bad]).all() and torch.isnan(dx[7]).any() and torch.isfinite(db).all()


@pytest.mark.parametrize("dtype,wdtype", [("bf16", "fp32"), ("fp32", "fp32")])
def test_autograd(dev, dtype, wdtype):
    from coat_amd.activation.norm import layer_norm, layer_norm_backward, layer_norm_forward
    x, dy, w, b = make(dev, 6 * 50, 520, TYPES[dtype], TYPES[wdtype], 2)
    x = x.view(6, 50, 520).requires_grad_()
    w.requires_grad_(), b.requires_grad_()
    y = layer_norm(x, w, b)
    y.backward(dy.view_as(y))
    with torch.no_grad():
        out = layer_norm_forward(x, w, b)
        grads = layer_norm_backward(dy.view_as(y), x, out[1], out[2], w)
        assert torch.equal(layer_norm(x, w, b), y) and torch.equal(out[0], y)
    for leaf, want in zip((x, w, b), grads):
        assert torch.equal(leaf.grad, want)
    x2 = x.detach().clone().requires_grad_()
    layer_norm(x2).backward(dy.view_as(y))  # without parameters
    check_backward(dy.view_as(y), x2.detach(), *layer_norm_forward(x2.detach())[1:], None, (x2.grad, None, None))
    w.grad = b.grad = None
    layer_norm(x.detach(), w, b).backward(dy.view_as(y))  # only the parameters
    assert torch.equal(w.grad, grads[1]) and torch.equal(b.grad, grads[2])


def test_gradient_against_differences(dev):
    """Central differences of sum(y * c) along random directions, in 64 bits around the kernel's own gradient."""
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    x, c, w, b = make(dev, 7, 300, torch.float32, torch.float32, 4)
    _, mean, rstd = layer_norm_forward(x, w, b, 1e-5)
    grads = layer_norm_backward(c, x, mean, rstd, w)
    g = torch.Generator().manual_seed(8)
    values = [t.double() for t in (x, w, b)]

    def f(vals):
        xd, wd, bd = vals
        n = (xd - xd.mean(1, keepdim=True)) * ((xd - xd.mean(1, keepdim=True)).square().mean(1, keepdim=True) + 1e-5).rsqrt()
        return ((n * wd + bd) * c.double()).sum().item()

    for k in range(3):
        d = torch.randn(values[k].shape, generator=g, dtype=torch.float64).to(dev)
        up, down = list(values), list(values)
        up[k], down[k] = values[k] + 1e-4 * d, values[k] - 1e-4 * d
        slope = (f(up) - f(down)) / 2e-4
        along = (grads[k].double() * d).sum().item()
        size = (grads[k].double().abs() * d.abs()).sum().item()
        assert abs(slope - along) <= 1e-5 * size, (k, slope, along)


def test_same_bits_twice_on_another_stream_and_from_a_graph(dev):
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    x, dy, w, b = make(dev, 2000, 1001, torch.bfloat16, torch.float32, 6)

    def step(x, dy):
        y, mean, rstd = layer_norm_forward(x, w, b)
        return (y, mean, rstd, *layer_norm_backward(dy, x, mean, rstd, w))

    want = step(x, dy)
    assert all(torch.equal(a, e) for a, e in zip(step(x, dy), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(other, want))
    sx, sdy = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sdy)
    for seed in (11, 12, 13):
        nx, ndy, _, _ = make(dev, 2000, 1001, torch.bfloat16, None, seed)
        sx.copy_(nx), sdy.copy_(ndy)
        graph.replay()
        eager = step(nx, ndy)  # the program's own work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, eager)), seed


def test_past_two_to_the_31_elements(dev):
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    M, N = (1 << 31) // 4096 + 64, 4096
    x = torch.zeros(M, N, dtype=torch.bfloat16, device=dev)
    tail = torch.randn(64, N, generator=torch.Generator().manual_seed(0)).bfloat16().to(dev)
    x[-64:] = tail
    w = torch.full((N,), 2.0, device=dev)
    y, mean, rstd = layer_norm_forward(x, w)
    want = layer_norm_forward(tail, w)
    assert torch.equal(y[-64:], want[0]) and torch.equal(mean[-64:], want[1]) and torch.equal(rstd[-64:], want[2])
    assert not y[:-64].any()
    dx, dw, db = layer_norm_backward(x, x, mean, rstd, w)
    part = layer_norm_backward(tail, tail, want[1], want[2], w)
    assert torch.equal(dx[-64:], part[0])
    check_backward(tail, tail, want[1], want[2], w, (None, dw, db))  # zero rows add nothing
