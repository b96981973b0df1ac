"""GPU: the AdamW step over many tensors with 32-bit states and the global gradient norm (qoptim_cuda.adamw_step_multi,
grad_norm_multi) against the formulas in 64 bits.

Bounds.  Hyperparameters are rounded once (2^-24 each); a moment takes three roundings on top: 6 * 2^-24 of the sum of its terms'
sizes.  The update takes a square root, a division and four more operations: 24 * 2^-24 of its terms' sizes, times lr; the new
parameter one rounding of its own type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HYPER = dict(beta1=0.9, beta2=0.999, lr=1e-3, wd=0.1, eps=1e-8)
E = 2.0 ** -24


def make(dev, sizes, pdtype, gdtype, master, seed, packed=False, fill=None):
    """Parallel lists params, grads, exp_avg, exp_avg_sq, masters: views of flat buffers, with guard elements between them."""
    g = torch.Generator().manual_seed(seed)
    gap = 1 if packed else 64

    def column(dtype, f):
        at, views = 1 if packed else 0, []
        flat = torch.full((sum(-(-n // gap) * gap + gap for n in sizes) + 2,), 7.0, dtype=dtype)
        for n in sizes:
            flat[at:at + n] = f(n).to(dtype)
            views.append((at, n))
            at += -(-n // gap) * gap + gap
        flat = flat.to(dev)
        return flat, [flat[a:a + n] for a, n in views]

    w = [torch.randn(n, generator=g) * 0.05 for n in sizes]
    it = iter(w)
    cols = {"params": column(pdtype, lambda n: next(it)), "grads": column(gdtype, lambda n: torch.randn(n, generator=g) * 1e-2),
            "exp_avg": column(torch.float32, lambda n: torch.randn(n, generator=g) * 1e-3),
            "exp_avg_sq": column(torch.float32, lambda n: torch.randn(n, generator=g).square() * 1e-5)}
    if master:
        it = iter(w)
        cols["masters"] = column(torch.float32, lambda n: next(it))
    return cols


def guards(flat, views):
    mask = torch.ones_like(flat, dtype=torch.bool)
    for v in views:
        mask[v.storage_offset():v.storage_offset() + v.numel()] = False
    return flat[mask]


def lists(cols):
    return {k: v[1] for k, v in cols.items()}


def step(cols, n, scale=None, **kw):
    from coat_amd.optimizer import qoptim_cuda
    c, h = lists(cols), {**HYPER, **kw}
    qoptim_cuda.adamw_step_multi(c["params"], c["grads"], c["exp_avg"], c["exp_avg_sq"], h["beta1"], h["beta2"], h["lr"], h["wd"], h["eps"],
                                 n, masters=c.get("masters"), grad_scale=scale)


def check_step(before, cols, n, scale=1.0, **kw):
    h = {**HYPER, **kw}
    c1, c2 = 1 - h["beta1"] ** n, math.sqrt(1 - h["beta2"] ** n)
    now = lists(cols)
    for i in range(len(now["params"])):
        old = {k: v[i].double() for k, v in before.items()}
        g = old["grads"] * scale
        w = old["masters"] if "masters" in old else old["params"]
        mt, vt = (h["beta1"] * old["exp_avg"], (1 - h["beta1"]) * g), (h["beta2"] * old["exp_avg_sq"], (1 - h["beta2"]) * g * g)
        m, v = sum(mt), sum(vt)
        denom = (v.sqrt() / c2 + h["eps"]) * c1
        update = m / denom + h["wd"] * w
        p = w - h["lr"] * update
        assert ((now["exp_avg"][i].double() - m).abs() <= 6 * E * (mt[0].abs() + mt[1].abs()) + 1e-38).all()
        assert ((now["exp_avg_sq"][i].double() - v).abs() <= 8 * E * v + 1e-38).all()
        bound = E * p.abs() + 24 * E * h["lr"] * ((mt[0].abs() + mt[1].abs()) / denom + h["wd"] * w.abs()) + 1e-38
        if "masters" in now:
            assert ((now["masters"][i].double() - p).abs() <= bound).all()
            assert torch.equal(now["params"][i], now["masters"][i].to(now["params"][i].dtype))
        else:
            half = torch.finfo(now["params"][i].dtype).eps / 2
            tiny = torch.finfo(now["params"][i].dtype).smallest_normal * half * 2
            assert ((now["params"][i].double() - p).abs() <= half * p.abs() * (1 + half) + bound + tiny).all()
        assert torch.equal(now["grads"][i], before["grads"][i])


SIZES = [1, 2, 7, 8, 9, 0, 63, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 100003]
KINDS = [("fp32", "fp32", False), ("bf16", "bf16", False), ("bf16", "fp32", True), ("bf16", "bf16", True), ("bf16", "fp32", False),
         ("fp16", "fp16", False), ("fp16", "fp32", True), ("fp16", "fp16", True), ("fp16", "fp32", False)]


@pytest.mark.parametrize("pd,gd,master", KINDS)
@pytest.mark.parametrize("packed", [False, True])
def test_step(dev, pd, gd, master, packed):
    cols = make(dev, SIZES, TYPES[pd], TYPES[gd], master, 1, packed)
    edges = {k: guards(*v).clone() for k, v in cols.items()}
    for n in (1, 2, 700):
        before = {k: [t.clone() for t in v[1]] for k, v in cols.items()}
        step(cols, n)
        check_step(before, cols, n)
    for k, v in cols.items():  # nothing beside the tensors is touched
        assert torch.equal(guards(*v), edges[k]), k


def test_more_tensors_than_a_launch_takes_and_bits_of_separate_calls(dev):
    sizes = [(37 * i) % 5000 for i in range(150)]
    together, apart = (make(dev, sizes, torch.float32, torch.float32, False, 2, True) for _ in range(2))
    step(together, 3)
    for i in range(len(sizes)):
        step({k: (v[0], v[1][i:i + 1]) for k, v in apart.items()}, 3)
    for k in together:
        assert torch.equal(together[k][0], apart[k][0]), k


def test_grad_scale_is_a_multiplication_of_the_gradients(dev):
    scale = torch.tensor(0.37, device=dev)
    cols = make(dev, SIZES, torch.bfloat16, torch.float32, True, 3)
    before = {k: [t.clone() for t in v[1]] for k, v in cols.items()}
    step(cols, 5, scale)
    check_step(before, cols, 5, scale.double().item())
    a, b = (make(dev, SIZES, torch.float32, torch.float32, False, 4) for _ in range(2))
    step(a, 2, torch.ones(1, device=dev))
    step(b, 2)
    assert all(torch.equal(a[k][0], b[k][0]) for k in a)


def test_zero_gradients_zero_states_and_values_that_are_not_finite(dev):
    cols = make(dev, [4100], torch.float32, torch.float32, False, 5)
    p, g, m, v = (cols[k][1][0] for k in ("params", "grads", "exp_avg", "exp_avg_sq"))
    g.zero_(), m.zero_(), v.zero_()
    old = p.clone()
    step(cols, 1)  # 0 / (0 + eps): only the decay is left
    assert ((p.double() - old.double() * (1 - 1e-3 * 0.1)).abs() <= 2 * E * old.double().abs()).all() and not m.any() and not v.any()
    step(cols, 2, wd=0.0)
    before = p.clone()
    step(cols, 3, wd=0.0)
    assert torch.equal(p, before)
    g[5], g[4099] = float("nan"), float("inf")
    step(cols, 4)
    bad = torch.zeros(4100, dtype=torch.bool, device=dev)
    bad[5] = bad[4099] = True
    assert torch.equal(~torch.isfinite(p), bad) and torch.isfinite(m[~bad]).all()


NORM_SIZES = [0, 1, 7, 8, 8191, 8192, 8193, 0, 70001]


@pytest.mark.parametrize("kinds", [("fp32",), ("bf16",), ("fp16",), ("bf16", "fp32", "fp16")])
@pytest.mark.parametrize("count", [1, 9, 300])
def test_grad_norm(dev, kinds, count):
    from coat_amd.optimizer import qoptim_cuda
    g = torch.Generator().manual_seed(count)
    flat = (torch.randn(200000, generator=g) * 0.01).to(dev)
    grads = [flat[i % 50 + 1:][:NORM_SIZES[(i + 1) % 9] if count > 1 else 70001].to(TYPES[kinds[i % len(kinds)]]) for i in range(count)]
    want = math.sqrt(sum((t.double() ** 2).sum().item() for t in grads))
    norm, none = qoptim_cuda.grad_norm_multi(grads)
    assert none is None and norm.dim() == 0 and norm.dtype == torch.float32
    assert abs(norm.item() - want) <= 2 * E * want
    for most in (want / 3, want * 3, 0.0):
        again, scale = qoptim_cuda.grad_norm_multi(grads, max_norm=most)
        s = min(1.0, most / (want + 1e-6))
        assert torch.equal(again, norm) and abs(scale.item() - s) <= 3 * E * s and (most < want or scale.item() == 1.0)


def test_grad_norm_of_a_large_tensor_slices_and_extremes(dev):
    from coat_amd.optimizer import qoptim_cuda
    big = torch.full((40_000_003,), 3e-4, device=dev)
    norm, _ = qoptim_cuda.grad_norm_multi([big, big[1:100], big[:0]])
    want = math.sqrt((40_000_003 + 99) * big[0].double().item() ** 2)
    assert abs(norm.item() - want) <= 2 * E * want
    huge = torch.full((1000,), 1e30, device=dev)  # squares beyond fp32
    assert abs(qoptim_cuda.grad_norm_multi([huge])[0].item() / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    small = torch.full((1000,), 1e-30, device=dev)
    assert abs(qoptim_cuda.grad_norm_multi([small])[0].item() / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    square = torch.randn(64, 64, device=dev)
    assert torch.allclose(qoptim_cuda.grad_norm_multi([square.t()])[0], square.norm(), rtol=1e-6)
    zero = torch.zeros(5, device=dev)
    norm, scale = qoptim_cuda.grad_norm_multi([zero], 1.0)
    assert norm.item() == 0.0 and scale.item() == 1.0
    norm, scale = qoptim_cuda.grad_norm_multi([zero[:0]], 1.0)
    assert norm.item() == 0.0 and scale.item() == 1.0
    zero[3] = float("inf")
    norm, scale = qoptim_cuda.grad_norm_multi([zero], 1.0)
    assert math.isinf(norm.item()) and scale.item() == 0.0
    zero[2] = float("nan")
    norm, scale = qoptim_cuda.grad_norm_multi([zero], 1.0)
    assert math.isnan(norm.item()) and math.isnan(scale.item())


def test_norm_and_step_on_another_stream_and_from_a_graph(dev):
    """The captured step keeps its step number and hyperparameters; gradients, states and the clipping follow the replays."""
    from coat_amd.optimizer import qoptim_cuda

    def clipped(cols):
        norm, scale = qoptim_cuda.grad_norm_multi(lists(cols)["grads"], max_norm=0.5)
        step(cols, 9, scale)
        return norm

    kinds = [300, 4097, 12345, 1]
    eager, other, graphed = (make(dev, kinds, torch.bfloat16, torch.bfloat16, True, 6) for _ in range(3))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clipped(graphed)
    side = torch.cuda.Stream()
    for k in range(4):
        new = make(dev, kinds, torch.bfloat16, torch.bfloat16, True, 60 + k)["grads"][0] * (k + 0.1)
        for cols in (eager, other, graphed):
            cols["grads"][0].copy_(new)
        graph.replay()
        want = clipped(eager)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            on_side = clipped(other)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(want, norm) and torch.equal(want, on_side)
        for key in eager:
            assert torch.equal(eager[key][0], graphed[key][0]) and torch.equal(eager[key][0], other[key][0]), (k, key)


def test_parameters_notice_that_they_were_written(dev):
    cols = make(dev, [100], torch.float32, torch.float32, False, 7)
    p = cols["params"][1][0] = cols["params"][1][0].clone().requires_grad_()
    y = (p * p).sum()
    with torch.no_grad():
        step(cols, 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_past_two_to_the_31_elements(dev):
    from coat_amd.optimizer import qoptim_cuda
    n, k = (1 << 31) + 5000, 6000
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device=dev) for _ in range(2))
    m, v = (torch.zeros(n, device=dev) for _ in range(2))
    tail = make(dev, [k], torch.bfloat16, torch.bfloat16, False, 8)
    for t, key in ((p, "params"), (g, "grads"), (m, "exp_avg"), (v, "exp_avg_sq")):
        t[-k:] = tail[key][1][0]
    norm, scale = qoptim_cuda.grad_norm_multi([g], max_norm=0.1)
    want, ws = qoptim_cuda.grad_norm_multi(tail["grads"][1], max_norm=0.1)
    assert torch.allclose(norm, want, rtol=2 * E, atol=0)  # the same squares in other groups
    qoptim_cuda.adamw_step_multi([p], [g], [m], [v], 0.9, 0.999, 1e-3, 0.1, 1e-8, 4, grad_scale=ws)
    step(tail, 4, ws)
    for t, key in ((p, "params"), (m, "exp_avg"), (v, "exp_avg_sq")):
        assert torch.equal(t[-k:], tail[key][1][0]) and not t[:-k].any(), key
