"""GPU: the operators beside the FP8 blocks where they are used: CoatAdamW with 32-bit states and clipping, the decoder layer's
attention with positions on several axes, and a training step of rotary, norm, gradient norm and step in one run."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

HYPER = (0.9, 0.95, 3e-3, 0.1, 1e-8)
E = 2.0 ** -24


def randn(dev, seed, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev)


# ------------------------------------------------------------------------------------------------ 8-bit states, scaled gradients
@pytest.mark.parametrize("expand", [False, True])
def test_scaled_steps_with_fp8_states_equal_steps_on_scaled_gradients(dev, expand):
    """fp32 tensors: the product of gradient and factor is the same fp32 number in the kernel as before it."""
    from coat_amd.optimizer import qoptim_cuda
    sizes = [1, 127, 128, 129, 1024, 5000, 0, 70001] + [33 * i for i in range(1, 40)]

    def state(seed):
        cols = {k: [] for k in ("p", "g", "m", "sm", "km", "cm", "v", "sv", "kv", "cv")}
        for i, n in enumerate(sizes):
            groups = (n + 127) // 128
            cols["p"].append(randn(dev, seed + i, n, scale=0.02))
            cols["g"].append(randn(dev, seed + 1000 + i, n, scale=1e-2))
            for k in "mv":
                cols[k].append(torch.zeros(n, dtype=torch.float8_e4m3fn, device=dev))
                cols["s" + k].append(torch.zeros(groups, device=dev))
                cols["k" + k].append(torch.ones(groups, device=dev))
                cols["c" + k].append(torch.ones(groups, device=dev))
        return cols

    def step(c, n, grads, scale):
        if expand:
            qoptim_cuda.fp8_adamw_expand_step_multi(c["p"], grads, c["m"], c["sm"], c["km"], c["cm"], c["v"], c["sv"], c["kv"], c["cv"],
                                                    *HYPER, n, 128, 16, grad_scale=scale)
        else:
            qoptim_cuda.fp8_adamw_step_multi(c["p"], grads, c["m"], c["sm"], c["v"], c["sv"], *HYPER, n, 128, grad_scale=scale)

    a, b = state(1), state(1)
    for n in (1, 2, 3):
        scale = torch.tensor(0.3 / n, device=dev)
        step(a, n, a["g"], scale)
        step(b, n, [g * scale for g in b["g"]], None)
    for k in a:
        for x, y in zip(a[k], b[k]):
            assert torch.equal(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x, y.view(torch.uint8) if y.dtype == torch.float8_e4m3fn else y), k
    with pytest.raises(RuntimeError, match="grad_scale"):
        step(a, 4, a["g"], torch.ones(1))


# ------------------------------------------------------------------------------------------------ CoatAdamW
def parameters(dev, dtype, seed, shapes):
    return [torch.nn.Parameter(randn(dev, seed + i, *s, scale=0.05, dtype=dtype)) for i, s in enumerate(shapes)]


def reference_step(w, m, v, g, n):
    beta1, beta2, lr, wd, eps = HYPER
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    denom = (v.sqrt() / (1 - beta2 ** n) ** 0.5 + eps) * (1 - beta1 ** n)
    return w - lr * (m / denom + wd * w), m, v


@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True), (torch.bfloat16, False)])
def test_optimizer_with_32_bit_states_and_clipping(dev, dtype, master):
    """Two groups, one of FP8 states; the 32-bit group against the formula in 64 bits, step by step from its own state."""
    from coat_amd.optimizer.fp8_adamw import CoatAdamW
    beta1, beta2, lr, wd, eps = HYPER
    norms, mats = parameters(dev, dtype, 1, [(64,), (513,), (7, 9)]), parameters(dev, dtype, 10, [(64, 64), (33, 5)])
    opt = CoatAdamW([dict(params=norms, state_bits=32, master_weights=master), dict(params=mats)], lr=lr, betas=(beta1, beta2), eps=eps,
                    weight_decay=wd, max_grad_norm=0.5)
    for n in (1, 2, 3):
        for i, p in enumerate(norms + mats):
            p.grad = randn(dev, 100 * n + i, *p.shape, scale=0.1, dtype=dtype)
        total = sum((p.grad.double() ** 2).sum() for p in norms + mats).sqrt().item()
        scale = min(1.0, 0.5 / (total + 1e-6))
        before = []
        for p in norms:
            s = opt.state[p]
            old = [torch.zeros_like(p).double()] * 2 if not s else [s["exp_avg"].double(), s["exp_avg_sq"].double()]
            before.append(((s["master"] if s and master else p.detach()).double().clone(), *[t.clone() for t in old]))
        grads = [p.grad.clone() for p in norms + mats]
        opt.step()
        assert abs(opt.grad_norm.item() - total) <= 2 * E * total
        assert all(torch.equal(p.grad, g) for p, g in zip(norms + mats, grads))  # the gradients stay as they were
        for p, (w, m, v) in zip(norms, before):
            s, g = opt.state[p], p.grad.double() * scale
            want, m1, v1 = reference_step(w, m, v, g, n)
            size = (beta1 * m).abs() + (1 - beta1) * g.abs()  # roundings as in the test of the step itself, 4 more in the factor
            assert s["exp_avg"].dtype == s["exp_avg_sq"].dtype == torch.float32 and int(s["step"]) == n
            assert ((s["exp_avg"].double() - m1).abs() <= 10 * E * size + 1e-38).all()
            assert ((s["exp_avg_sq"].double() - v1).abs() <= 16 * E * v1 + 1e-38).all()
            denom = (v1.sqrt() / (1 - beta2 ** n) ** 0.5 + eps) * (1 - beta1 ** n)
            bound = E * want.abs() + 36 * E * lr * (size / denom + wd * w.abs()) + 1e-38
            held = s["master"] if master else p.detach()
            half = 0.0 if held.dtype == torch.float32 else torch.finfo(held.dtype).eps / 2
            assert ((held.double() - want).abs() <= bound + half * (want.abs() + bound)).all()
            if master:
                assert torch.equal(p.detach(), held.to(dtype))
        for p in mats:
            assert opt.state[p]["exp_avg"].dtype == torch.float8_e4m3fn


def test_optimizer_clips_fp8_states_with_the_same_factor(dev):
    """The FP8-state group of a clipping optimizer, bit for bit the multi-tensor step with the factor of the gradient norm."""
    from coat_amd.optimizer import qoptim_cuda
    from coat_amd.optimizer.fp8_adamw import CoatAdamW
    beta1, beta2, lr, wd, eps = HYPER
    shapes = [(64, 64), (33, 5), (1000,)]
    a, b = parameters(dev, torch.float32, 3, shapes), parameters(dev, torch.float32, 3, shapes)
    kw = dict(lr=lr, betas=(beta1, beta2), eps=eps, weight_decay=wd)
    clipped, plain = CoatAdamW(a, **kw, max_grad_norm=0.1), CoatAdamW(b, **kw)
    for n in (1, 2):
        for i, (x, y) in enumerate(zip(a, b)):
            x.grad = randn(dev, 50 * n + i, *x.shape, scale=0.1)
        scale = qoptim_cuda.grad_norm_multi([x.grad for x in a], 0.1)[1]
        assert scale.item() < 1.0
        for x, y in zip(a, b):
            y.grad = x.grad * scale
        clipped.step(), plain.step()
        for x, y in zip(a, b):
            assert torch.equal(x, y)
            for k, t in clipped.state[x].items():
                u = plain.state[y][k]
                assert torch.equal(t.view(torch.uint8), u.view(torch.uint8)) if t.dtype == torch.float8_e4m3fn else torch.equal(t, u), k


def test_optimizer_state_dict_round_trip_and_late_masters(dev):
    from coat_amd.optimizer.fp8_adamw import CoatAdamW
    p, q = parameters(dev, torch.bfloat16, 5, [(300,)])[0], parameters(dev, torch.bfloat16, 5, [(300,)])[0]
    first = CoatAdamW([p], lr=1e-2, state_bits=32, master_weights=True, max_grad_norm=1.0)
    second = CoatAdamW([q], lr=1e-2, state_bits=32, master_weights=True, max_grad_norm=1.0)
    for n in range(2):
        p.grad = randn(dev, n, 300, dtype=torch.bfloat16)
        first.step()
    saved = copy.deepcopy(first.state_dict())
    with torch.no_grad():
        q.copy_(p)
    second.load_state_dict(saved)
    assert second.state[q]["master"].dtype == torch.float32 and second.param_groups[0]["state_bits"] == 32
    p.grad, q.grad = (randn(dev, 9, 300, dtype=torch.bfloat16) for _ in range(2))
    first.step(), second.step()
    assert torch.equal(p, q) and all(torch.equal(first.state[p][k], second.state[q][k]) for k in ("exp_avg", "exp_avg_sq", "master", "step"))
    # a state without masters, continued with them: the copy starts from the parameter
    r = parameters(dev, torch.bfloat16, 6, [(40,)])[0]
    opt = CoatAdamW([dict(params=[r], state_bits=32)])
    r.grad = randn(dev, 1, 40, dtype=torch.bfloat16)
    opt.step()
    opt.param_groups[0]["master_weights"] = True
    old = r.detach().float()
    opt.step()
    assert torch.equal(opt.state[r]["master"].bfloat16(), r) and (opt.state[r]["master"] - old).abs().max() <= 1.2e-3  # lr (1 + wd |w|)
    # FP8 states are not taken for 32-bit ones
    opt8 = CoatAdamW([r])
    opt8.step()
    opt8.param_groups[0]["state_bits"] = 32
    with pytest.raises(RuntimeError, match="exp_avg must all be torch.float32"):
        opt8.step()


# ------------------------------------------------------------------------------------------------ attention with several axes
def attention_module(dev, **kw):
    from coat_amd.models.coat_llama import CoatLlamaConfig, LlamaSdpaAttentionWithoutLinear
    config = CoatLlamaConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=256, **kw)
    return LlamaSdpaAttentionWithoutLinear(config)


def test_attention_turns_by_positions_of_several_axes(dev):
    from coat_amd.models._attention import sdpa
    from coat_amd.models.rotary import RotaryAxes, rotary_axes
    B, S = 2, 96
    pos = torch.randint(0, 1000, (3, B, S), generator=torch.Generator().manual_seed(1)).to(dev)
    leaves = [randn(dev, i, B, S, n, dtype=torch.bfloat16).requires_grad_() for i, n in ((2, 512), (3, 256), (4, 256))]
    module = attention_module(dev, rotary_sections=(16, 24, 24)).train()
    out = module(*leaves, position_ids=pos)[0]
    g = randn(dev, 5, B, S, 512, dtype=torch.bfloat16)
    grads = torch.autograd.grad(out, leaves, g)
    q, k = rotary_axes(leaves[0].view(B, S, 4, 128), leaves[1].view(B, S, 2, 128), pos, RotaryAxes(128, (16, 24, 24)))
    k, v = (t.transpose(1, 2).repeat_interleave(2, dim=1) for t in (k, leaves[2].view(B, S, 2, 128)))
    want = sdpa(q.transpose(1, 2), k, v, is_causal=True).transpose(1, 2).reshape(B, S, 512)
    assert torch.equal(out, want)
    for a, e in zip(grads, torch.autograd.grad(want, leaves, g)):
        assert torch.equal(a, e)
    shared = module(*leaves, position_ids=pos[:, :1])[0]  # positions of one sequence for the batch
    assert torch.equal(shared, module(*leaves, position_ids=pos[:, :1].expand(3, B, S))[0])
    with pytest.raises(ValueError, match="rotary_sections"):
        attention_module(dev)(*leaves, position_ids=pos)
    # one axis of positions still takes the one-axis rotary
    flat = torch.arange(S, device=dev).expand(B, S)
    assert torch.equal(module(*leaves, position_ids=flat)[0], attention_module(dev).train()(*leaves, position_ids=flat)[0])


def test_decoder_layer_trains_with_positions_of_several_axes(dev):
    """The whole FP8 layer: forward and backward run, and change where only the positions change."""
    from coat_amd.activation.real_quantization import Coat_quantize_bgn, Coat_quantize_end
    from coat_amd.models.coat_llama import CoatLlamaConfig, CoatLlamaDecoderLayer
    from coat_amd.utils._fp8manager import FP8Manager
    FP8Manager.is_first_microbatch = True
    torch.manual_seed(0)
    config = CoatLlamaConfig(hidden_size=256, intermediate_size=512, num_attention_heads=2, rotary_sections=(16, 24, 24), coat_fp8_args=dict(group_size=16))
    layer = CoatLlamaDecoderLayer(config, 0).to(dev).bfloat16().train()
    begin, end = Coat_quantize_bgn(layer.qargs), Coat_quantize_end(layer.qargs)
    x = randn(dev, 1, 2, 64, 256, dtype=torch.bfloat16).requires_grad_()
    outs = []
    for far in (1, 50, 50):
        pos = torch.randint(0, far, (3, 2, 64), generator=torch.Generator().manual_seed(2)).to(dev)
        y = end(*layer(*begin(x), position_ids=pos)[0])
        grad = torch.autograd.grad(y.float().square().mean(), x)[0]
        assert torch.isfinite(y).all() and torch.isfinite(grad).all() and grad.any()
        outs.append((y, grad))
    assert not torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[1][0], outs[2][0]) and torch.equal(outs[1][1], outs[2][1])


# ------------------------------------------------------------------------------------------------ a training step
def small_model(x, wq, wk, nw, nb, pos, rotate, norm):
    """Rotated q and k, plain attention with x as values, the last norm, a loss."""
    B, S, D = x.shape
    q, k = rotate((x @ wq).view(B, S, 4, 32), (x @ wk).view(B, S, 4, 32), pos)
    p = ((q.transpose(1, 2) @ k.transpose(1, 2).transpose(2, 3).contiguous()) / 32 ** 0.5).softmax(-1)
    o = (p @ x.view(B, S, 4, D // 4).transpose(1, 2).contiguous()).transpose(1, 2).reshape(B, S, D)
    return norm(o, nw, nb).square().mul(0.1).exp().mean()


def test_training_step_of_all_operators_against_64_bits(dev):
    """Gradients and stepped parameters of rotary, attention, norm, global norm and AdamW in fp32 against the same in 64 bits.  Each of
    some eight operations in a row is off by at most 256 roundings of 2^-24 of the size of what it computes: 1.2e-4 of a
    gradient's 2-norm; the step moves a parameter by at most about lr, in the gradient's sign, so parameters are compared where
    the gradient is well clear of zero."""
    from coat_amd.activation.norm import layer_norm
    from coat_amd.models.rotary import RotaryAxes, rotary_axes
    from coat_amd.optimizer.fp8_adamw import CoatAdamW
    B, S, D = 2, 50, 128
    plan = RotaryAxes(32, (4, 6, 6))
    x, pos = randn(dev, 1, B, S, D), torch.randint(0, 200, (3, B, S), generator=torch.Generator().manual_seed(2)).to(dev)
    start = [randn(dev, 3, D, 128, scale=0.1), randn(dev, 4, D, 128, scale=0.1), 1 + randn(dev, 5, D, scale=0.1), randn(dev, 6, D, scale=0.1)]
    own = [torch.nn.Parameter(t.clone()) for t in start]
    small_model(x, *own, pos, lambda q, k, p: rotary_axes(q, k, p, plan), layer_norm).backward()

    def rotate(q, k, p):
        ang = torch.cat([p[a].double()[..., None] * 10000.0 ** -(torch.arange(f, f + n, dtype=torch.float64, device=dev) / 16)
                         for a, f, n in ((0, 0, 4), (1, 4, 6), (2, 10, 6))], -1)[:, :, None]
        c, s = ang.cos(), ang.sin()
        return [torch.cat((t[..., :16] * c - t[..., 16:] * s, t[..., 16:] * c + t[..., :16] * s), -1) for t in (q, k)]

    def norm(t, w, b):
        t = t - t.mean(-1, keepdim=True)
        return t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w + b

    ref = [t.double().requires_grad_() for t in start]
    small_model(x.double(), *ref, pos, rotate, norm).backward()
    for a, e in zip(own, ref):
        assert (a.grad.double() - e.grad).norm() <= 1.2e-4 * e.grad.norm()
    opt = CoatAdamW([dict(params=own, state_bits=32)], lr=1e-3, betas=(0.9, 0.95), weight_decay=0.1, max_grad_norm=1e-3)
    opt.step()
    total = sum((e.grad ** 2).sum() for e in ref).sqrt()
    assert abs(opt.grad_norm.item() - total.item()) <= 1.2e-4 * total.item()
    for a, e, s in zip(own, ref, start):
        g = e.grad * min(1.0, 1e-3 / (total.item() + 1e-6))
        want = s.double() - 1e-3 * (g / (g.abs() + 1e-8) + 0.1 * s.double())  # the first step: m / sqrt(v) is the sign
        clear = e.grad.abs() > 0.05 * e.grad.norm() / e.grad.numel() ** 0.5
        # g / (|g| + eps) moves by eps / |g| of itself per relative change of g
        assert clear.float().mean() > 0.9 and ((a.double() - want).abs()[clear] <= 1e-6 + E * want.abs()[clear] * 4).all()


def test_training_step_captured_and_replayed(dev):
    """The functional calls of a step in one graph, replayed on new inputs next to eager steps of the same start."""
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_backward, rotary_axes_forward
    from coat_amd.optimizer import qoptim_cuda
    B, S, H, D = 2, 40, 4, 64
    plan = RotaryAxes(D, (8, 12, 12))

    def make():
        w = randn(dev, 1, H * D, dtype=torch.bfloat16) + 1
        return dict(w=w, b=randn(dev, 2, H * D, dtype=torch.bfloat16), mw=w.float(), mb=randn(dev, 2, H * D, dtype=torch.bfloat16).float(),
                    m=[torch.zeros(H * D, device=dev) for _ in range(2)], v=[torch.zeros(H * D, device=dev) for _ in range(2)])

    def run(s, x, pos, dy):
        q, _ = rotary_axes_forward(x, None, pos, plan)
        y, mean, rstd = layer_norm_forward(q.flatten(2), s["w"], s["b"])
        dx, dw, db = layer_norm_backward(dy, q.flatten(2), mean, rstd, s["w"])
        dq, _ = rotary_axes_backward(dx.view_as(x), None, pos, plan)
        norm, scale = qoptim_cuda.grad_norm_multi([dw, db], 0.5)
        qoptim_cuda.adamw_step_multi([s["w"], s["b"]], [dw, db], s["m"], s["v"], 0.9, 0.95, 1e-2, 0.1, 1e-8, 5, masters=[s["mw"], s["mb"]],
                                     grad_scale=scale)
        return y, dq, norm

    def inputs(seed):
        return (randn(dev, seed, B, S, H, D, dtype=torch.bfloat16), torch.randint(0, 99, (3, B, S), generator=torch.Generator().manual_seed(seed)).to(dev),
                randn(dev, seed + 1, B, S, H * D, dtype=torch.bfloat16))

    eager, graphed, static = make(), make(), [t.clone() for t in inputs(10)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(graphed, *static)
    for seed in (20, 30, 40, 50):
        new = inputs(seed)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        want = run(eager, *new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, want)), seed
        for k in eager:
            for a, e in zip(*[t if isinstance(t, list) else [t] for t in (graphed[k], eager[k])]):
                assert torch.equal(a, e), (seed, k)


def test_autograd_of_rotary_and_norm_captured_and_replayed(dev):
    """Forward and backward through autograd inside one capture, with leaves of the graph's own; eager runs on other leaves."""
    from coat_amd.activation.norm import layer_norm
    from coat_amd.models.rotary import RotaryAxes, rotary_axes
    plan = RotaryAxes(64, (8, 12, 12))

    def run(x, w, b, pos, g):
        q, k = rotary_axes(x, x[:, :, :2], pos, plan)
        y = layer_norm(torch.cat((q, k), 2).flatten(2), w, b)
        return (y, *torch.autograd.grad(y, (x, w, b), g))

    def inputs(seed):
        return [randn(dev, seed, 2, 30, 4, 64, dtype=torch.bfloat16).requires_grad_(), (1 + randn(dev, seed + 1, 384, scale=0.1)).requires_grad_(),
                randn(dev, seed + 2, 384).requires_grad_(), torch.randint(0, 99, (3, 2, 30), generator=torch.Generator().manual_seed(seed)).to(dev),
                randn(dev, seed + 3, 2, 30, 384, dtype=torch.bfloat16)]

    static = inputs(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*static)
    for seed in (10, 20, 30):
        new = inputs(seed)
        with torch.no_grad():
            for a, e in zip(static, new):
                a.copy_(e)
        graph.replay()
        want = run(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, want)), seed


def test_two_threads_on_streams_of_their_own(dev):
    import threading

    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    from coat_amd.optimizer import qoptim_cuda

    def work(seed):
        x, w = randn(dev, seed, 300, 1001, dtype=torch.bfloat16), randn(dev, seed + 1, 1001)
        m, v = torch.zeros_like(w), torch.zeros_like(w)
        for n in range(1, 20):
            y, mean, rstd = layer_norm_forward(x, w, w)
            dx, dw, db = layer_norm_backward(y, x, mean, rstd, w)
            norm, scale = qoptim_cuda.grad_norm_multi([dw, db], 1.0)
            qoptim_cuda.adamw_step_multi([w], [dw], [m], [v], *HYPER, n, grad_scale=scale)
        return y, dx, w, m, v, norm

    want, got = [work(1), work(50)], [None, None]
    torch.cuda.synchronize()

    def thread(i, seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = work(seed)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=thread, args=(i, s)) for i, s in enumerate((1, 50))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, e in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, e))
