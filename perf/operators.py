"""Timing cases of the streaming passes that a training step has beside its FP8 blocks: LayerNorm (forward, and backward with the
reduction of the weight's and the bias's gradient), rotary positions with several axes (forward and backward, q and k together),
and the AdamW step over many tensors with 32-bit states, clipped by the global norm of the gradients.

``own`` false: the operators as elementary torch operations in 32 bits, rounded once at the end (angles of far positions and long
sums in 64).  ``own`` true: the package's entry points.  ``exact``: the definitions in 64 bits, written apart from the plain form."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_HYPER = (0.9, 0.95, 3e-4, 0.1, 1e-8, 12)  # beta1, beta2, lr, weight decay, eps, step number


# ------------------------------------------------------------------------------------------------------------- the cases
def listed():
    """Sizes: hidden 4096 / 5120, heads 32 / 40 of 128, 4 x 2048 tokens, intermediate 11008 and vocabulary 32000 are those of the
    repository's decoder layers and loss; the others are generic."""
    return [
        # the hidden states of four positions, as when a handful of tokens is scored: launch latency
        dict(name="ln_fwd_4x4096_bf16", op="ln", direction="fwd", rows=4, cols=4096, dtype="bf16", weight="bf16", bias=True, sliced=False),
        # the last norm before the head over a whole batch, forward and backward
        dict(name="ln_fwd_8192x4096_bf16", op="ln", direction="fwd", rows=8192, cols=4096, dtype="bf16", weight="bf16", bias=True, sliced=False),
        dict(name="ln_bwd_8192x4096_bf16", op="ln", direction="bwd", rows=8192, cols=4096, dtype="bf16", weight="fp32", bias=True, sliced=False),
        # ragged: packed sequences of an odd total, an odd width, half precision with fp32 weights, x a column slice of a wider tensor
        dict(name="ln_bwd_1531x1001_fp16", op="ln", direction="bwd", rows=1531, cols=1001, dtype="fp16", weight="fp32", bias=True, sliced=True),
        # a norm over each head of q: very many short rows, weight without bias
        dict(name="ln_bwd_262144x128_bf16", op="ln", direction="bwd", rows=262144, cols=128, dtype="bf16", weight="bf16", bias=False, sliced=False),
        # one token: latency
        dict(name="rot_fwd_1x1_bf16", op="rot", direction="fwd", batch=1, seq=1, heads=32, kv_heads=32, dim=128, sections="16,24,24",
             restart=False, pairs=False, dtype="bf16", far=40000, fused=False),
        # a batch of image / video / text tokens with time, height and width positions
        dict(name="rot_fwd_4x2048_bf16", op="rot", direction="fwd", batch=4, seq=2048, heads=32, kv_heads=32, dim=128, sections="16,24,24",
             restart=False, pairs=False, dtype="bf16", far=4096, fused=True),
        # its gradient with grouped heads
        dict(name="rot_bwd_4x2048_bf16", op="rot", direction="bwd", batch=4, seq=2048, heads=40, kv_heads=8, dim=128, sections="16,24,24",
             restart=False, pairs=False, dtype="bf16", far=4096, fused=False),
        # image patches in fp32: two axes with frequencies of their own, neighbouring pairs, an unrotated rest, odd length
        dict(name="rot_fwd_3x1021_fp32", op="rot", direction="fwd", batch=3, seq=1021, heads=12, kv_heads=12, dim=80, sections="16,16",
             restart=True, pairs=True, dtype="fp32", far=1024, fused=False),
        # the norm weights of a 32-layer model (two a layer and the last): latency
        dict(name="adamw_65_norms_fp32", op="adamw", sizes="4096*65", dtype="fp32", grads="fp32", master=False, clip=1.0, packed=False),
        # bf16 parameters of odd sizes with fp32 masters, laid out one after the other without padding
        dict(name="adamw_ragged_bf16_master", op="adamw", sizes="1*3,127*4,4099*9,120001*12,1500007*8", dtype="bf16", grads="bf16",
             master=True, clip=1.0, packed=True),
        # one decoder layer and the embedding
        dict(name="adamw_333M_fp32", op="adamw", sizes="4096*2,16777216*4,45088768*3,131072000", dtype="fp32", grads="fp32", master=False,
             clip=1.0, packed=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("ln", "ln", "rot", "rot", "adamw", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "ln":
        cols = _log(rng, 24, 16384)
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        weight = rng.choice((dtype, "fp32", "none"))
        return dict(op="ln", direction=rng.choice(("fwd", "bwd")), rows=_log(rng, 1, max(2, min(262144, (1 << 25) // cols))), cols=cols, dtype=dtype,
                    weight=weight, bias=weight != "none" and rng.random() < 0.7, sliced=rng.random() < 0.3)
    if op == "rot":
        dim = rng.choice((32, 64, 80, 96, 128, 256))
        heads, kv_heads = rng.choice(((1, 1), (4, 0), (8, 2), (12, 12), (14, 2), (32, 32), (32, 8), (40, 40), (64, 8)))
        left, sections = dim // 2 - (rng.randrange(0, dim // 8) if rng.random() < 0.4 else 0), []
        for axis in range(rng.randint(1, 4) - 1):
            sections.append(rng.randint(1, max(1, left // 2)))
            left -= sections[-1]
        sections.append(left)
        batch = rng.randint(1, 4)
        most = min(4096, (1 << 26) // (batch * (heads + kv_heads) * dim))
        return dict(op="rot", direction=rng.choice(("fwd", "bwd")), batch=batch, seq=_log(rng, 1, most), heads=heads, kv_heads=kv_heads, dim=dim,
                    sections=",".join(map(str, sections)), restart=rng.random() < 0.4, pairs=rng.random() < 0.4, dtype=dtype,
                    far=_log(rng, 16, 1 << 20), fused=rng.random() < 0.4)
    count = _log(rng, 1, 200)
    most = max(2, min(1 << 24, (1 << 27) // count))
    sizes = [_log(rng, 1, most) for _ in range(min(count, 12))]
    each = count // len(sizes)
    return dict(op="adamw", sizes=",".join("%d*%d" % (s, each) for s in sizes), dtype=dtype, grads=rng.choice((dtype, "fp32")),
                master=dtype != "fp32" and rng.random() < 0.6, clip=rng.choice((0.0, 1.0, 1e6)), packed=rng.random() < 0.4)


def _sizes(case):
    parts = [p.split("*") for p in case["sizes"].split(",")]
    return [int(p[0]) for p in parts for _ in range(int(p[1]) if len(p) > 1 else 1)]


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _bytes(kind):
    return 0 if kind == "none" else 4 if kind == "fp32" else 2


def work(case):
    if case["op"] == "ln":
        n, e, w = case["rows"] * case["cols"], _bytes(case["dtype"]), _bytes(case["weight"]) * case["cols"]
        if case["direction"] == "fwd":
            return {"bytes": 2 * n * e + w * (1 + case["bias"]) + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": 3 * n * e + w * (2 + case["bias"]) + 8 * case["rows"], "flops": 14 * n}
    if case["op"] == "rot":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * _bytes(case["dtype"]) + 8 * tokens * len(_sections(case)), "flops": 3 * n}
    n = sum(_sizes(case))
    return {"bytes": n * (16 + _bytes(case["grads"]) + 2 * 4 * case["master"] + _bytes(case["dtype"]) * (1 if case["master"] else 2)), "flops": 16 * n}


# ------------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    state, dtype = {"case": case}, _TYPES[case["dtype"]]
    if case["op"] == "ln":
        M, N = case["rows"], case["cols"]

        def rows(t):  # a tensor of its own, or the middle columns of a wider one
            t = t.to(dtype)
            if not case["sliced"]:
                return t
            wide = torch.zeros(M, 2 * N + 13, dtype=dtype, device="cuda")
            wide[:, 5:5 + N] = t
            return wide[:, 5:5 + N]

        state["x"] = rows(randn(M, N) * (0.5 + 1.5 * torch.rand(M, 1, generator=gen, device="cuda")) + 0.3 * randn(M, 1) + 0.1)
        state["w"] = None if case["weight"] == "none" else (1 + 0.2 * randn(N)).to(_TYPES[case["weight"]])
        state["b"] = (0.1 * randn(N)).to(state["w"].dtype) if case["bias"] else None
        state["eps"] = 1e-5
        if case["direction"] == "bwd":
            xd = state["x"].double()
            mean = xd.mean(1)
            state["mean"], state["rstd"] = mean.float(), ((xd - mean[:, None]).square().mean(1) + 1e-5).rsqrt().float()
            state["dy"] = rows(1e-2 * randn(M, N))
        return state
    if case["op"] == "rot":
        B, S, H, K, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        if case["fused"]:  # q and k are slices of one projection's output, which holds v too
            qkv = randn(B, S, (H + 2 * max(K, 1)) * D).to(dtype)
            state["q"] = qkv[..., :H * D].view(B, S, H, D)
            state["k"] = qkv[..., H * D:(H + K) * D].view(B, S, K, D) if K else None
        else:
            state["q"], state["k"] = randn(B, S, H, D).to(dtype), randn(B, S, K, D).to(dtype) if K else None
        sections = _sections(case)
        state["positions"] = torch.randint(0, case["far"], (len(sections), B, S), generator=gen, device="cuda")
        state["theta"] = 10000.0
        if own:
            from coat_amd.models.rotary import RotaryAxes
            state["plan"] = RotaryAxes(D, sections, theta=10000.0, restart=case["restart"], pairs=case["pairs"])
        else:
            state["freq"], state["axis"] = (t.cuda() for t in _frequencies(case, 10000.0))
        return state
    sizes = _sizes(case)
    at, end = [], 0  # where each tensor begins in its flat buffer
    for n in sizes:
        at.append(end)
        end += n if case["packed"] else -(-n // 64) * 64
    master = case["master"]
    w = randn(end) * 0.02
    state["params"] = w.to(dtype)
    state["masters"] = w if master else None
    state["exp_avg"] = randn(end) * 1e-3
    state["exp_avg_sq"] = randn(end).square() * 1e-6
    state["grads"] = (randn(end) * 2e-3).to(_TYPES[case["grads"]])
    for key in ("params", "masters", "exp_avg", "exp_avg_sq", "grads"):
        state[key + "_list"] = None if state[key] is None else [state[key][a:a + n] for a, n in zip(at, sizes)]
    return state


def _frequencies(case, theta):
    """Radians a position, in 64 bits, and the axis of each pair."""
    sections = _sections(case)
    total = sum(sections)
    axis = torch.cat([torch.full((n,), a, dtype=torch.int64) for a, n in enumerate(sections)])
    index = torch.cat([torch.arange(n, dtype=torch.float64) / n for n in sections]) if case["restart"] else torch.arange(total, dtype=torch.float64) / total
    return theta ** -index, axis


# ------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "ln":
        return _ln_forward(state) if case["direction"] == "fwd" else _ln_backward(state)
    return _rotary(state) if case["op"] == "rot" else _adamw(state)


def _ln_forward(state):
    x, w, b, eps = (state[k] for k in ("x", "w", "b", "eps"))
    if own:
        from coat_amd.activation.norm import layer_norm_forward
        return layer_norm_forward(x, w, b, eps)
    xf = x.float()
    mean = xf.mean(1, keepdim=True)
    c = xf - mean
    rstd = (c.square().mean(1, keepdim=True) + eps).rsqrt()
    y = c * rstd
    if w is not None:
        y = y * w.float()
    if b is not None:
        y = y + b.float()
    return y.to(x.dtype), mean.squeeze(1), rstd.squeeze(1)


def _ln_backward(state):
    x, w, dy, mean, rstd = (state[k] for k in ("x", "w", "dy", "mean", "rstd"))
    if own:
        from coat_amd.activation.norm import layer_norm_backward
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w, bias_grad=state["b"] is not None)
    else:
        g, n = dy.float(), (x.float() - mean[:, None]) * rstd[:, None]
        dw = (g * n).sum(0).to(w.dtype) if w is not None else None
        db = g.sum(0).to(w.dtype) if state["b"] is not None else None
        if w is not None:
            g = g * w.float()
        dx = ((g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True)) * rstd[:, None]).to(x.dtype)
    return [t for t in (dx, dw, db) if t is not None]


def _rotary(state):
    case, q, k = state["case"], state["q"], state["k"]
    inverse = case["direction"] == "bwd"
    if own:
        from coat_amd.models.rotary import rotary_axes_backward, rotary_axes_forward
        q, k = (rotary_axes_backward if inverse else rotary_axes_forward)(q, k, state["positions"], state["plan"])
        return [q] if k is None else [q, k]
    angle = state["positions"][state["axis"]].permute(1, 2, 0).double() * state["freq"]  # [B, S, pairs]
    c, s = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    if inverse:
        s = -s

    def turn(t):
        f, n = t.float(), 2 * c.shape[-1]
        a, b = (f[..., 0:n:2], f[..., 1:n:2]) if case["pairs"] else (f[..., :n // 2], f[..., n // 2:n])
        u, v = a * c - b * s, b * c + a * s
        out = torch.stack((u, v), -1).flatten(-2) if case["pairs"] else torch.cat((u, v), -1)
        return torch.cat((out, f[..., n:]), -1).to(t.dtype)

    return [turn(t) for t in (q, k) if t is not None]


def _adamw(state):
    clip = state["case"]["clip"]
    beta1, beta2, lr, wd, eps, step = _HYPER
    p, w, m, v, g = (state[k + "_list"] for k in ("params", "masters", "exp_avg", "exp_avg_sq", "grads"))
    norm = scale = None
    if own:
        from coat_amd.optimizer import qoptim_cuda
        if clip:
            norm, scale = qoptim_cuda.grad_norm_multi(g, max_norm=clip)
        qoptim_cuda.adamw_step_multi(p, g, m, v, beta1, beta2, lr, wd, eps, step, masters=w, grad_scale=scale)
    else:
        g32 = [t.float() for t in g]
        if clip:
            norm = torch.stack([t.sum(dtype=torch.float64) for t in torch._foreach_mul(g32, g32)]).sum().sqrt().float()
            g32 = torch._foreach_mul(g32, (clip / (norm + 1e-6)).clamp(max=1.0))
        p32 = w if w is not None else [t.float() for t in p]
        torch._foreach_mul_(m, beta1)
        torch._foreach_add_(m, g32, alpha=1 - beta1)
        torch._foreach_mul_(v, beta2)
        torch._foreach_add_(v, torch._foreach_mul(g32, g32), alpha=1 - beta2)
        denom = torch._foreach_sqrt(v)
        torch._foreach_div_(denom, math.sqrt(1 - beta2 ** step))
        torch._foreach_add_(denom, eps)
        torch._foreach_mul_(denom, 1 - beta1 ** step)
        update = torch._foreach_div(m, denom)
        torch._foreach_add_(update, p32, alpha=wd)
        torch._foreach_add_(p32, update, alpha=-lr)
        if p32 is not p:
            torch._foreach_copy_(p, p32)
    out = [state["params"], state["exp_avg"], state["exp_avg_sq"]]
    return out + [t for t in (state["masters"], norm) if t is not None]


# ------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ln":
        x = s["x"].double()
        w = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if s["w"] is None else s["w"].double()
        if case["direction"] == "fwd":
            mean = x.sum(1) / x.shape[1]
            var = (x - mean[:, None]).pow(2).sum(1) / x.shape[1]
            rstd = 1 / torch.sqrt(var + s["eps"])
            y = (x - mean[:, None]) * (rstd[:, None] * w)
            return (y if s["b"] is None else y + s["b"].double()), mean, rstd
        mean, rstd, dy = s["mean"].double(), s["rstd"].double(), s["dy"].double()
        hat = (x - mean[:, None]) * rstd[:, None]
        t = dy * w
        dx = rstd[:, None] * (t - (t.sum(1, keepdim=True) + hat * (t * hat).sum(1, keepdim=True)) / x.shape[1])
        return [dx] + ([(dy * hat).sum(0)] if s["w"] is not None else []) + ([dy.sum(0)] if s["b"] is not None else [])
    if case["op"] == "rot":
        sections = _sections(case)
        pos = s["positions"].double()
        total, sign, angles = sum(sections), -1.0 if case["direction"] == "bwd" else 1.0, []
        first = 0
        for a, n in enumerate(sections):
            for i in range(n):
                e = i / n if case["restart"] else (first + i) / total
                angles.append(pos[a] * 10000.0 ** -e)
            first += n
        z = torch.polar(torch.ones((), dtype=torch.float64, device=pos.device), sign * torch.stack(angles, -1))[:, :, None]
        outs = []
        for t in (s["q"], s["k"]):
            if t is None:
                continue
            d = t.double()
            lo, hi = (slice(0, 2 * total, 2), slice(1, 2 * total, 2)) if case["pairs"] else (slice(0, total), slice(total, 2 * total))
            r = torch.complex(d[..., lo].contiguous(), d[..., hi].contiguous()) * z
            out = d.clone()
            out[..., lo], out[..., hi] = r.real, r.imag
            outs.append(out)
        return outs
    beta1, beta2, lr, wd, eps, step = _HYPER
    sizes, clip = _sizes(case), case["clip"]
    flat = {k: (None if s[k] is None else s[k].double()) for k in ("params", "masters", "exp_avg", "exp_avg_sq", "grads")}
    used = torch.zeros(flat["params"].numel(), dtype=torch.bool, device="cuda")
    at = 0
    for n in sizes:
        used[at:at + n] = True
        at += n if case["packed"] else -(-n // 64) * 64
    g = flat["grads"] * used
    norm = None
    if clip:
        norm = torch.sqrt((g * g).sum())
        g = g * torch.clamp(clip / (norm + 1e-6), max=1.0)
    w = flat["masters"] if case["master"] else flat["params"]
    m = beta1 * flat["exp_avg"] + (1 - beta1) * g
    v = beta2 * flat["exp_avg_sq"] + (1 - beta2) * g ** 2
    new = w * (1 - lr * wd) - lr * (m / (1 - beta1 ** step)) / (torch.sqrt(v / (1 - beta2 ** step)) + eps)
    # eps is added before the first moment's correction, which divides both: the same quotient
    w, m, v = torch.where(used, new, w), torch.where(used, m, flat["exp_avg"]), torch.where(used, v, flat["exp_avg_sq"])
    out = [torch.where(used, w, flat["params"]), m, v]
    return out + ([w] if case["master"] else []) + ([norm] if norm is not None else [])
