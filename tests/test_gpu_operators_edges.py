"""GPU: LayerNorm, multi-axis rotary, gradient norm and 32-bit AdamW at the edges of what they promise."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def randn(dev, seed, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev)


# ------------------------------------------------------------------------------------------------ what torch cannot see
@pytest.mark.parametrize("grad", [False, True])
def test_traced_functions_follow_their_inputs(dev, grad):
    from coat_amd.activation.norm import layer_norm
    from coat_amd.models.rotary import RotaryAxes, rotary_axes
    plan, pos = RotaryAxes(32, (6, 10)), torch.arange(5, device=dev).expand(2, 1, 5)
    w = randn(dev, 1, 32)

    def f(x):
        return layer_norm(rotary_axes(x, None, pos, plan)[0], w)

    a, b = (randn(dev, s, 1, 5, 3, 32).requires_grad_(grad) for s in (2, 3))
    traced = torch.jit.trace(f, (a,), check_trace=False)
    for x in (b, a):
        assert torch.equal(traced(x), f(x))


def test_tangents_are_refused(dev):
    import torch.autograd.forward_ad as fwAD

    from coat_amd.activation.norm import layer_norm
    from coat_amd.models.rotary import RotaryAxes, rotary_axes
    plan, pos = RotaryAxes(32, (6, 10)), torch.arange(5, device=dev).expand(2, 1, 5)
    x = randn(dev, 2, 1, 5, 3, 32)
    with fwAD.dual_level():
        for grad in (False, True):
            d = fwAD.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x))
            with pytest.raises(NotImplementedError):
                layer_norm(d)
            with pytest.raises(NotImplementedError):
                rotary_axes(d, None, pos, plan)
        assert torch.equal(layer_norm(x), layer_norm(x.clone()))


# ------------------------------------------------------------------------------------------------ rotary plans
def test_loaded_and_copied_modules_rotate_as_before(dev):
    import copy
    import io

    from coat_amd.models.coat_llama import CoatLlamaConfig, LlamaSdpaAttentionWithoutLinear
    module = LlamaSdpaAttentionWithoutLinear(CoatLlamaConfig(hidden_size=256, num_attention_heads=2, rotary_sections=(16, 24, 24))).eval()
    x = [randn(dev, s, 1, 20, 256, dtype=torch.bfloat16) for s in (1, 2, 3)]
    pos = torch.randint(0, 50, (3, 1, 20), generator=torch.Generator().manual_seed(4)).to(dev)
    want = module(*x, position_ids=pos)[0]
    for where in ("cpu", dev):
        buffer = io.BytesIO()
        torch.save(module, buffer)
        buffer.seek(0)
        loaded = torch.load(buffer, map_location=where, weights_only=False)
        for other in (loaded, copy.deepcopy(loaded)):
            assert all(t.device == d for d, pair in other.rotary_axes._tables.items() for t in pair)
            assert torch.equal(other(*x, position_ids=pos)[0], want)


def test_tables_of_another_device_are_refused(dev):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    plan, q, pos = RotaryAxes(32, (6, 10)), randn(dev, 1, 1, 5, 2, 32), torch.arange(5, device=dev).expand(2, 1, 5)
    turns, axis = plan.tables(q.device)
    for bad in ((turns.cpu(), axis), (turns, axis.cpu())):
        plan._tables[q.device] = bad
        with pytest.raises(ValueError, match="tables"):
            rotary_axes_forward(q, None, pos, plan)


def test_a_plan_may_be_dropped_while_another_stream_still_reads_its_tables(dev):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes, rotary_axes_forward
    q, pos = randn(dev, 1, 1, 50, 4, 128).requires_grad_(), torch.arange(50, device=dev).expand(3, 1, 50)
    want = rotary_axes_forward(q, None, pos, RotaryAxes(128, (16, 24, 24)))[0]
    work, side = randn(dev, 2, 4096, 4096), torch.cuda.Stream()
    torch.cuda.synchronize()
    plan = RotaryAxes(128, (16, 24, 24))
    addresses = {t.data_ptr() for t in plan.tables(q.device)}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            work = (work @ work).clamp_(-1, 1)  # the rotation waits behind this
        out = rotary_axes(q, None, pos, plan)[0]
        out.backward(want.detach(), retain_graph=False)
    del plan
    other = [torch.full((64,), 7.5, dtype=torch.float64, device=dev) for _ in range(200)] + [torch.full((64,), 1, dtype=torch.int32, device=dev) for _ in range(200)]
    assert not side.query() and not addresses & {t.data_ptr() for t in other}  # not handed out again while that work is queued
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert torch.allclose(q.grad, q, rtol=1e-5, atol=1e-5)  # turned there and back


def test_more_tokens_than_a_launch_takes_blocks_in_a_row(dev):
    """2^24 + 5000 tokens whose 520 pairs leave one token to a block; three tokens of a time are compared with their own calls."""
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    S, D = (1 << 24) + 5000, 1040
    plan = RotaryAxes(D, (200, 320))
    base = randn(dev, 1, 1, 7, 1, D, dtype=torch.bfloat16)
    q = torch.as_strided(base, (1, S, 1, D), (7 * D, 0, D, 1))  # the same token everywhere: no 35 GB of input
    pos = torch.arange(S, device=dev).expand(2, 1, S)
    out = rotary_axes_forward(q, None, pos, plan)[0]
    for at in (0, 5, (1 << 24) - 3, (1 << 24) + 2000, S - 3):
        assert torch.equal(out[:, at:at + 3], rotary_axes_forward(q[:, :3], None, pos[:, :, at:at + 3], plan)[0]), at
    assert torch.isfinite(out.view(-1)[::997]).all()


def test_plans_made_and_dropped_around_a_capture(dev):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    q, pos = randn(dev, 1, 1, 9, 2, 128), torch.arange(9, device=dev).expand(3, 1, 9)
    plan, other = RotaryAxes(128, (16, 24, 24)), RotaryAxes(128, (16, 24, 24), theta=500.0)
    rotary_axes_forward(q, None, pos, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_axes_forward(q, None, pos, plan)[0]
        del other
    for k in range(3):
        q.copy_(randn(dev, 5 + k, 1, 9, 2, 128))
        graph.replay()
        assert torch.equal(out, rotary_axes_forward(q, None, pos, plan)[0])
    del graph, plan
    fresh = [torch.zeros(64, dtype=torch.float64, device=dev) for _ in range(50)]
    torch.cuda.synchronize()
    want = rotary_axes_forward(q, None, pos, RotaryAxes(128, (16, 24, 24)))[0]
    assert torch.equal(out, want) and not any(t.any() for t in fresh)


# ------------------------------------------------------------------------------------------------ LayerNorm
def test_parameter_gradients_of_more_columns_than_a_launch_takes_blocks_in_a_row(dev):
    """One row of 2^27 + 100 columns: each gradient is one product, or dy itself, with the roundings of the separate torch operations."""
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    N = (1 << 27) + 100
    x, dy = (torch.randn(1, N, generator=torch.Generator(dev).manual_seed(s), device=dev) for s in (1, 2))
    w = torch.ones(N, device=dev)
    _, mean, rstd = layer_norm_forward(x, w)
    assert abs(mean.item()) < 1e-3 and abs(rstd.item() - 1) < 1e-3
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w)
    h = (x - mean) * rstd
    assert torch.equal(db, dy[0]) and torch.equal(dw, (dy * h)[0]) and torch.isfinite(dx).all()
    only = layer_norm_backward(dy, x, mean, rstd, w, False, x_grad=False)
    assert torch.equal(only[1], dw) and only[0] is only[2] is None


@pytest.mark.parametrize("M,N", [(3, 8193), (20, 8200), (5, 10239), (7, 10241), (9, 12288), (40, 13712), (300, 14337), (2, 16384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_frozen_parameters_do_not_change_the_bits_of_dx(dev, M, N, dtype):
    """Rows that are held in four pieces a lane with the sums of the parameters' gradients, and in two without."""
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    x, dy, w = randn(dev, 1, M, N, dtype=dtype), randn(dev, 2, M, N, dtype=dtype), 1 + randn(dev, 3, N, scale=0.2)
    _, mean, rstd = layer_norm_forward(x, w)
    want = layer_norm_backward(dy, x, mean, rstd, w)[0]
    for weight, bias in ((False, False), (True, False), (False, True)):
        assert torch.equal(layer_norm_backward(dy, x, mean, rstd, w, bias, weight_grad=weight)[0], want), (weight, bias)


@pytest.mark.parametrize("M,N", [(400, 100), (400, 500), (400, 1000), (400, 4096), (400, 5000), (300, 12000), (300, 20000), (200, 40001)])
def test_rows_far_from_zero_keep_their_mean_to_the_last_bits(dev, M, N):
    """fp32 rows around m = 1000 with a spread of about 1.  In the mean square over the rows, with u = 2^-24, an error at most as large as
    the sum it belongs to and uniformly distributed: the additions of a tree take (1 + 1/2 + 1/4 ...) / 3 <= 2/3 of (u m)^2, 16 wave sums
    one after the other (rows beyond 16384) 1.95 of it, the product 1/3, a rounded 1/N at most 1 in every row alike (a division has
    none): at most 1.52 u m, with a tenth more for the sample 1.7.  The deviations are off by that, and by at most 20 roundings of
    themselves (8 squares a piece, two pieces and 13 operations, half of it after the root; then the last three)."""
    from coat_amd.activation.norm import layer_norm_forward
    x = randn(dev, N, M, N) * (0.5 + torch.rand(M, 1, generator=torch.Generator().manual_seed(1)).to(dev)) + 1000.0
    y, mean, rstd = layer_norm_forward(x, None, None, 1e-5)
    xd, u = x.double(), 2.0 ** -24
    m = xd.mean(1)
    d = xd - m[:, None]
    r = (d.square().mean(1) + 1e-5).rsqrt()
    rms = lambda t: t.square().mean().sqrt()  # noqa: E731
    assert rms(mean.double() - m) <= 1.7 * u * rms(m), rms(mean.double() - m) / (u * rms(m))
    off = y.double() / r[:, None] - d
    assert rms(off) <= u * (1.7 * rms(m) + 20 * rms(d)), rms(off) / (u * (1.7 * rms(m) + 20 * rms(d)))
    assert ((rstd.double() / r - 1).abs() <= (20 + N / 1024) * u + (4 * u * m * r) ** 2).all()


# ------------------------------------------------------------------------------------------------ rotary in fp32
def test_angles_of_fp32_heads_lose_nothing_to_the_rounded_argument(dev):
    """Heads (1, 0) return cosine and sine themselves.  Bound on how far the angle they stand for is off, in the mean square: two
    roundings of at most 2^-25 each (the library's result and its correction), uniformly distributed, the library's taken one and a
    half times as large: sqrt(1 + 1.5^2) 2^-25 / sqrt(3) = 3.1e-8 radians.  An argument rounded to fp32 is off by up to 2^-26 of a turn
    where it is a quarter turn or more: 5.4e-8 in the mean square by itself."""
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_backward, rotary_axes_forward
    plan, S = RotaryAxes(128, (30, 34), theta=500.0), 20000
    q = torch.zeros(1, S, 1, 128, device=dev)
    q[..., :64] = 1.0
    pos = torch.randint(0, 1 << 20, (2, 1, S), generator=torch.Generator().manual_seed(1)).to(dev)
    freq = torch.tensor([500.0 ** -(j / 64) for j in range(64)], dtype=torch.float64, device=dev)
    ang = pos[[0] * 30 + [1] * 34].permute(1, 2, 0).double()[:, :, None] * freq
    for f, sign in ((rotary_axes_forward, 1.0), (rotary_axes_backward, -1.0)):
        out = f(q, None, pos, plan)[0].double()
        off = out[..., 64:] * sign * ang.cos() - out[..., :64] * ang.sin()
        far = ang.cos() < 0  # at least a quarter turn from a whole one
        assert off[far].square().mean().sqrt() <= 3.25 ** 0.5 * 2.0 ** -25 / 3 ** 0.5, off[far].square().mean().sqrt()
        assert off.square().mean().sqrt() <= 3.25 ** 0.5 * 2.0 ** -25 / 3 ** 0.5, off.square().mean().sqrt()
