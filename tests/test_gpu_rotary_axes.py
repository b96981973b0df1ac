"""GPU: rotary positions with several axes (coat_amd.models.rotary) against the rotation in 64 bits.

Bounds.  u = half a step of the output's type.  The fraction of a turn is rounded to fp32 (at most 2^-26 of a turn, 1e-7 radians),
sine and cosine are good to 2^-22, each product and the sum round by 2^-24: 5e-7 (|x1| + |x2|) covers them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def angles(pos, sections, theta, restart):
    total, out, first = sum(sections), [], 0
    for a, n in enumerate(sections):
        for i in range(n):
            out.append(pos[a].double() * theta ** -(i / n if restart else (first + i) / total))
        first += n
    return torch.stack(out, -1)[:, :, None]  # [B, S, 1, pairs]


def rotated(x, pos, sections, theta, restart, pairs, sign=1.0):
    """(the rotation in 64 bits, |x1| + |x2| of each element's pair)."""
    P = sum(sections)
    ang = angles(pos, sections, theta, restart) * sign
    lo, hi = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if pairs else (slice(0, P), slice(P, 2 * P))
    d = x.double()
    out, size = d.clone(), torch.zeros_like(d)
    out[..., lo] = d[..., lo] * ang.cos() - d[..., hi] * ang.sin()
    out[..., hi] = d[..., hi] * ang.cos() + d[..., lo] * ang.sin()
    size[..., lo] = size[..., hi] = d[..., lo].abs() + d[..., hi].abs()
    return out, size


def check(x, got, pos, plan, sign=1.0):
    want, size = rotated(x, pos, plan.sections, plan.theta, plan.restart, plan.pairs, sign)
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() + 5e-7 * size + torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps / 2 * (size > 0)
    err = (got.double() - want).abs()
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert (err <= bound).all(), (err - bound).max()


def randn(dev, seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def positions(dev, seed, axes, B, S, far):
    return torch.randint(0, far, (axes, B, S), generator=torch.Generator().manual_seed(seed)).to(dev)


CASES = [  # batch, seq, heads, kv_heads, head_dim, sections
    (1, 1, 1, 1, 2, (1,)), (1, 1, 32, 32, 128, (16, 24, 24)), (2, 5, 4, 2, 64, (8, 12, 12)), (3, 17, 3, 1, 80, (16, 16)),
    (1, 33, 14, 2, 96, (5, 0, 43)), (2, 9, 2, 2, 72, (9, 7, 3)), (1, 130, 8, 8, 128, (64,)), (2, 3, 5, 5, 50, (3, 4, 5, 6)),
    (1, 3, 2, 1, 256, (40, 44, 44)), (1, 2, 1, 1, 1000, (200, 300)), (1, 2, 2, 1, 2048, (1024,)), (4, 300, 12, 4, 64, (10, 11, 11))]


@pytest.mark.parametrize("B,S,H,K,D,sections", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("restart,pairs", [(False, False), (True, True), (False, True), (True, False)])
def test_forward_and_backward(dev, B, S, H, K, D, sections, dtype, restart, pairs):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_backward, rotary_axes_forward
    plan = RotaryAxes(D, sections, theta=10000.0, restart=restart, pairs=pairs)
    q, k = randn(dev, 1, B, S, H, D, dtype=TYPES[dtype]), randn(dev, 2, B, S, K, D, dtype=TYPES[dtype])
    pos = positions(dev, 3, len(sections), B, S, 5000)
    for f, sign in ((rotary_axes_forward, 1.0), (rotary_axes_backward, -1.0)):
        qo, ko = f(q, k, pos, plan)
        check(q, qo, pos, plan, sign)
        check(k, ko, pos, plan, sign)
    only, none = rotary_axes_forward(q, None, pos, plan)
    assert none is None and torch.equal(only, rotary_axes_forward(q, k, pos, plan)[0])
    none, only = rotary_axes_forward(None, k, pos, plan)
    assert none is None and torch.equal(only, rotary_axes_forward(q, k, pos, plan)[1])


@pytest.mark.parametrize("far", [1 << 20, 1 << 40])
def test_far_and_negative_positions(dev, far):
    """fp32 tensors: an angle that had been taken in 32 bits would be off by far * 2^-24 radians.  At 2^40 the product of position
    and frequency itself is rounded to 2^-15 of a turn in 64 bits: the reference there starts from the same rounded product."""
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    plan = RotaryAxes(64, (10, 10, 12), theta=1e6)
    q = randn(dev, 4, 2, 40, 3, 64)
    pos = positions(dev, 5, 3, 2, 40, far) - far // 2
    got = rotary_axes_forward(q, None, pos, plan)[0]
    if far <= 1 << 20:
        check(q, got, pos, plan)
    turns, axis = plan.tables(dev)
    t = pos[axis.long()].permute(1, 2, 0).double() * turns
    ang = ((t - t.round()) * 2 * torch.pi)[:, :, None]
    a, b = q.double()[..., :32], q.double()[..., 32:]
    want = torch.cat((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()), -1)
    size = (a.abs() + b.abs()).repeat(1, 1, 1, 2)
    assert ((got.double() - want).abs() <= 2.0 ** -24 * want.abs() + 5e-7 * size).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("D,sections,pairs", [(128, (16, 24, 24), False), (70, (9, 10, 11), False), (70, (9, 10, 11), True)])
def test_slices_transposes_and_broadcasts_give_the_same_bits(dev, dtype, D, sections, pairs):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    plan = RotaryAxes(D, sections, pairs=pairs)
    B, S, H, K = 2, 37, 6, 2
    qkv = randn(dev, 6, B, S, (H + 2 * K) * D + 1, dtype=TYPES[dtype])[..., 1:]  # an odd first element
    q, k = qkv[..., :H * D].unflatten(-1, (H, D)), qkv[..., H * D:(H + K) * D].unflatten(-1, (K, D))
    pos = positions(dev, 7, len(sections), B, S, 900)
    want = rotary_axes_forward(q.contiguous(), k.contiguous(), pos, plan)
    check(q, want[0], pos, plan)
    forms = [(q, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(0, 1).contiguous().transpose(0, 1)),
             (q.transpose(2, 3).contiguous().transpose(2, 3), k)]
    for form in forms:
        for a, e in zip(rotary_axes_forward(*form, pos, plan), want):
            assert torch.equal(a, e)
    shared = pos[:, :1]  # one row of positions for the batch, as a broadcast and as a strided view of [B, S, axes]
    want = rotary_axes_forward(q, k, shared.expand(-1, B, S).contiguous(), plan)
    for p in (shared, shared.expand(-1, B, S), shared.permute(1, 2, 0).contiguous().permute(2, 0, 1), shared.int()):
        for a, e in zip(rotary_axes_forward(q, k, p, plan), want):
            assert torch.equal(a, e)
    heads = rotary_axes_forward(q[:, :, :1].expand(B, S, H, D), None, pos, plan)[0]  # one head for all
    assert torch.equal(heads, rotary_axes_forward(q[:, :, :1], None, pos, plan)[0].expand(B, S, H, D))


def test_one_axis_and_a_zero_position(dev):
    """Equal positions on every axis are the one-axis rotary; position 0 changes nothing."""
    from coat_amd.models.coat_llama import fused_rotary
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    plan = RotaryAxes(128, (16, 24, 24))
    q = randn(dev, 8, 2, 70, 4, 128, dtype=torch.bfloat16)
    same = torch.arange(70, device=dev).expand(3, 2, 70)
    got = rotary_axes_forward(q, None, same, plan)[0]
    old = fused_rotary(q.flatten(2), 4, 128, 10000.0).transpose(1, 2)
    # the one-axis tables hold fp32 angles: 70 * 2^-24 radians, next to one rounding on each side
    size = (q.float()[..., :64].abs() + q.float()[..., 64:].abs()).repeat(1, 1, 1, 2)
    assert ((got.float() - old.float()).abs() <= 2.0 ** -8 * (got.float().abs() + old.float().abs()) + 1e-5 * size).all()
    assert torch.equal(rotary_axes_forward(q, None, torch.zeros_like(same), plan)[0], q)


def test_values_that_are_not_finite_stay_in_their_pair(dev):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    for pairs, other in ((False, 3 + 30), (True, 2)):
        plan = RotaryAxes(64, (10, 20), pairs=pairs)
        q = randn(dev, 9, 1, 4, 2, 64)
        q[0, 1, 1, 3], q[0, 2, 0, 63] = float("nan"), float("inf")
        out = rotary_axes_forward(q, None, positions(dev, 1, 2, 1, 4, 50) + 1, plan)[0]
        bad = torch.zeros_like(q, dtype=torch.bool)
        bad[0, 1, 1, 3] = bad[0, 1, 1, other] = True
        assert torch.equal(torch.isnan(out), bad) and torch.isinf(out[0, 2, 0, 63]) and torch.isinf(out).sum() == 1


def test_empty(dev):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    plan = RotaryAxes(32, (8, 8))
    for B, S in ((0, 5), (2, 0)):
        q, k = torch.empty(B, S, 4, 32, device=dev), torch.empty(B, S, 2, 32, device=dev)
        qo, ko = rotary_axes_forward(q, k, torch.empty(2, B, S, dtype=torch.int64, device=dev), plan)
        assert qo.shape == q.shape and ko.shape == k.shape
    q = torch.empty(2, 3, 0, 32, device=dev)
    assert rotary_axes_forward(q, None, torch.zeros(2, 2, 3, dtype=torch.int64, device=dev), plan)[0].shape == q.shape


def test_autograd_and_differences(dev):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes, rotary_axes_backward
    plan = RotaryAxes(48, (6, 8, 10), pairs=True)
    q, k = randn(dev, 1, 2, 11, 4, 48).requires_grad_(), randn(dev, 2, 2, 11, 2, 48).requires_grad_()
    pos = positions(dev, 3, 3, 2, 11, 300)
    gq, gk = randn(dev, 4, 2, 4, 11, 48).transpose(1, 2), randn(dev, 5, 2, 11, 2, 48)  # a gradient in attention's layout
    qo, ko = rotary_axes(q, k, pos, plan)
    torch.autograd.backward((qo, ko), (gq, gk))
    want = rotary_axes_backward(gq, gk, pos, plan)
    assert torch.equal(q.grad, want[0]) and torch.equal(k.grad, want[1])
    for x, g, grad in ((q, gq, q.grad), (k, gk, k.grad)):
        d = randn(dev, 6, *x.shape).double()
        f = lambda v: (rotated(v, pos, plan.sections, plan.theta, False, True)[0] * g.double()).sum().item()  # noqa: E731
        slope = (f(x.detach().double() + 1e-3 * d) - f(x.detach().double() - 1e-3 * d)) / 2e-3
        assert abs(slope - (grad.double() * d).sum().item()) <= 1e-6 * (grad.double() * d).abs().sum().item()
    q.grad = None
    rotary_axes(q, k, pos, plan)[0].backward(gq)  # k's result unused
    assert torch.equal(q.grad, want[0])
    out, none = rotary_axes(q, None, pos, plan)
    assert none is None and torch.equal(out, qo)
    q.grad, fixed = None, k.detach()
    qo, ko = rotary_axes(q, fixed, pos, plan)  # k is no leaf of the graph
    torch.autograd.backward((qo, ko), (gq, gk))
    assert torch.equal(q.grad, want[0]) and fixed.grad is None


def test_c_entry_ignores_the_pointers_of_no_heads(dev):
    from coat_amd import _hip
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    plan = RotaryAxes(32, (8, 8))
    x, pos = randn(dev, 7, 2, 5, 3, 32), positions(dev, 8, 2, 2, 5, 100)
    turns, axis = plan.tables(x.device)
    want, out = rotary_axes_forward(x, None, pos, plan)[0], torch.empty_like(x)
    one, none = (x.data_ptr(), out.data_ptr(), 5 * 96, 96, 32, 3), (1, 3, 0, 0, 0, 0)
    for args in (one + none, none + one):
        out.zero_()
        assert _hip.lib().coat_rope_axes(*args, _hip.F32, pos.data_ptr(), 10, 5, 1, 2, turns.data_ptr(), axis.data_ptr(), 16, 32, 0, 0, 2, 5,
                                         _hip.stream(x.device)) == 0
        assert torch.equal(out, want)


def test_another_stream_and_a_graph(dev):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_backward, rotary_axes_forward
    plan = RotaryAxes(128, (16, 24, 24))

    def make(seed):
        return (randn(dev, seed, 2, 100, 8, 128, dtype=torch.bfloat16), randn(dev, seed + 1, 2, 100, 2, 128, dtype=torch.bfloat16),
                positions(dev, seed + 2, 3, 2, 100, 4000))

    def step(q, k, pos):
        a, b = rotary_axes_forward(q, k, pos, plan)
        return (a, b, *rotary_axes_backward(a, b, pos, plan))

    first = make(20)
    want = step(*first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*first)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    static = [t.clone() for t in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for seed in (30, 40, 50):
        new = make(seed)
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        eager = step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, eager)), seed


def test_past_two_to_the_31_elements(dev):
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    plan = RotaryAxes(128, (16, 24, 24))
    S = (1 << 31) // (64 * 128) + 8
    q = torch.zeros(1, S, 64, 128, dtype=torch.bfloat16, device=dev)
    tail = randn(dev, 3, 1, 8, 64, 128, dtype=torch.bfloat16)
    q[:, -8:] = tail
    pos = torch.arange(S, device=dev).expand(3, 1, S)
    out = rotary_axes_forward(q, None, pos, plan)[0]
    assert torch.equal(out[:, -8:], rotary_axes_forward(tail, None, pos[:, :, -8:], plan)[0]) and not out[:, :-8].any()
