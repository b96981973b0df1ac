"""CPU: refusals of LayerNorm, multi-axis rotary, gradient norm and 32-bit AdamW, at the C entries and in Python."""
import ctypes

import pytest
import torch

EINVAL, ESHAPE, EDTYPE, EALIGN = -1, -2, -3, -5


@pytest.fixture(scope="module")
def L():
    from coat_amd import _hip
    return _hip.lib()


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096)
    p.keep = buf
    return (ctypes.addressof(buf) + 15) & ~15


def test_layer_norm_entries(L, p):
    f, b = L.coat_layer_norm_forward, L.coat_layer_norm_backward
    assert f(p, 0, 7, p, p, 0, p, p, p, 4, 64, 1e-5, None) == EDTYPE
    assert f(p, 0, 0, p, p, 5, p, p, p, 4, 64, 1e-5, None) == EDTYPE
    assert f(p, 0, 0, None, p, 0, p, p, p, 4, 64, 1e-5, None) == EINVAL      # a bias without a weight
    assert f(p, 0, 0, p, p, 0, p, p, p, 4, 0, 1e-5, None) == EINVAL          # no columns
    assert f(p, 0, 0, p, p, 0, p, p, p, -1, 64, 1e-5, None) == EINVAL
    assert f(p, 0, 0, p, p, 0, p, p, p, 4, 64, -1e-5, None) == EINVAL
    assert f(p, 0, 0, p, p, 0, p, p, p, 4, 64, float("nan"), None) == EINVAL
    assert f(p, 32, 0, p, p, 0, p, p, p, 4, 64, 1e-5, None) == ESHAPE        # pitch < columns
    assert f(None, 0, 0, p, p, 0, p, p, p, 4, 64, 1e-5, None) == EINVAL
    assert f(p, 0, 0, p, p, 0, p, None, p, 4, 64, 1e-5, None) == EINVAL
    assert f(p + 2, 0, 0, p, p, 0, p, p, p, 4, 64, 1e-5, None) == EALIGN     # fp32 at an address of 2 mod 4
    assert f(p, 0, 1, p + 1, p, 1, p, p, p, 4, 64, 1e-5, None) == EALIGN
    assert f(None, 0, 0, None, None, 0, None, None, None, 0, 64, 1e-5, None) == 0
    assert L.coat_layer_norm_partials(-1, 4) == EINVAL and L.coat_layer_norm_partials(4, 0) == EINVAL
    assert all(1 <= L.coat_layer_norm_partials(M, N) <= 65535 for M in (0, 1, 5, 1000, 10 ** 9) for N in (1, 4096, 10 ** 6))
    assert b(p, 0, p, 0, 9, p, p, p, 0, p, p, p, p, 4, 4, 64, None) == EDTYPE
    assert b(p, 0, p, 0, 0, p, p, p, 9, p, p, p, p, 4, 4, 64, None) == EDTYPE
    assert b(p, 0, p, 0, 0, p, p, None, 0, p, p, p, p, 4, 4, 64, None) == EINVAL     # dw without a weight
    assert b(p, 0, p, 0, 0, p, p, p, 0, p, p, p, None, 4, 4, 64, None) == EINVAL     # no workspace
    assert b(p, 0, p, 0, 0, p, p, p, 0, p, p, p, p, 0, 4, 64, None) == EINVAL
    assert b(p, 0, p, 0, 0, p, p, p, 0, p, p, p, p, 65536, 4, 64, None) == EINVAL
    assert b(None, 0, p, 0, 0, p, p, p, 0, p, p, p, p, 4, 4, 64, None) == EINVAL
    assert b(p, 0, p, 63, 0, p, p, p, 0, p, p, p, p, 4, 4, 64, None) == ESHAPE
    assert b(p, 63, p, 0, 0, p, p, p, 0, p, p, p, p, 4, 4, 64, None) == ESHAPE
    assert b(p, 0, p, 0, 0, p, p, p, 0, p + 1, p, p, p, 4, 4, 64, None) == EALIGN
    assert b(p, 0, p, 0, 0, p, p, p, 0, p, p, p, p, 4, 4, (1 << 31) + 1, None) == ESHAPE
    assert b(p, 0, p, 0, 0, p, p, p, 0, None, None, None, None, 0, 4, 64, None) == 0  # nothing wanted


def rope(L, p, **kw):
    a = dict(q=p, qo=p, qb=64, qs=64, qh=32, heads=2, k=p, ko=p, kb=64, ks=64, kh=32, kheads=1, dt=0, pos=p, pa=1, pb=1, ps=1, axes=2,
             turns=p, axis=p, pairs=16, dim=32, adjacent=0, inverse=0, batch=1, seq=1)
    a.update(kw)
    return L.coat_rope_axes(*a.values(), None)


def test_rope_axes_entry(L, p):
    assert rope(L, p, dt=3) == EDTYPE
    for bad in (dict(batch=-1), dict(seq=-1), dict(heads=-1), dict(kheads=-1), dict(axes=0), dict(pairs=0), dict(dim=1), dict(adjacent=2),
                dict(inverse=2), dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(pos=None), dict(turns=None), dict(axis=None)):
        assert rope(L, p, **bad) == EINVAL, bad
    for bad in (dict(pairs=17), dict(dim=2049), dict(heads=1025), dict(kheads=1025), dict(batch=1 << 40, seq=1), dict(batch=1 << 40, seq=1 << 40)):
        assert rope(L, p, **bad) == ESHAPE, bad
    for bad in (dict(q=p + 2), dict(ko=p + 1), dict(pos=p + 4), dict(turns=p + 4), dict(axis=p + 2)):
        assert rope(L, p, **bad) == EALIGN, bad
    assert rope(L, p, batch=0) == 0 and rope(L, p, seq=0) == 0 and rope(L, p, heads=0, kheads=0) == 0


def test_grad_norm_entries(L, p):
    i64, i32, vp = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p
    n, d, g = (i64 * 2)(100, 8193), (i32 * 2)(0, 1), (vp * 2)(p, p)
    assert L.coat_grad_norm_partials(2, n) == 3 and L.coat_grad_norm_partials(0, None) == 0
    assert L.coat_grad_norm_partials(1, (i64 * 1)(1 << 33)) == 2048
    assert L.coat_grad_norm_partials(2, (i64 * 2)(5, -1)) == EINVAL and L.coat_grad_norm_partials(1, None) == EINVAL
    assert L.coat_grad_norm_partials(1, (i64 * 1)(1 << 62)) == ESHAPE
    f = L.coat_grad_norm_multi
    assert f(-1, g, d, n, 1.0, p, 3, p, None) == EINVAL
    assert f(2, g, d, n, 1.0, p, 2, p, None) == EINVAL                      # workspace too small
    assert f(2, g, d, n, 1.0, None, 3, p, None) == EINVAL
    assert f(2, g, d, n, 1.0, p, 3, None, None) == EINVAL
    assert f(2, g, d, n, -1.0, p, 3, p, None) == EINVAL
    assert f(2, g, d, n, float("nan"), p, 3, p, None) == EINVAL
    assert f(2, (vp * 2)(p, None), d, n, 1.0, p, 3, p, None) == EINVAL
    assert f(2, g, (i32 * 2)(0, 4), n, 1.0, p, 3, p, None) == EDTYPE
    assert f(2, (vp * 2)(p + 2, p), d, n, 1.0, p, 3, p, None) == EALIGN
    assert f(2, g, d, n, 1.0, p + 4, 3, p, None) == EALIGN


def test_adamw_step_entry(L, p):
    i64, vp, f = ctypes.c_int64, ctypes.c_void_p, L.coat_adamw_step_multi
    n, a, h = (i64 * 2)(100, 10), (vp * 2)(p, p), (ctypes.c_double * 5)(0.9, 0.999, 1e-3, 0.1, 1e-8)
    none, odd = (vp * 2)(p, None), (vp * 2)(p, p + 2)
    assert f(-1, a, 0, a, 0, a, a, None, n, h, 1, None, None) == EINVAL
    assert f(0, None, 0, None, 0, None, None, None, None, None, 1, None, None) == 0
    assert f(2, a, 0, a, 0, a, a, None, n, h, 0, None, None) == EINVAL        # steps count from 1
    assert f(2, a, 0, a, 0, a, a, None, n, None, 1, None, None) == EINVAL
    for bad in ((1.0, 0.9), (0.9, 1.0), (-0.1, 0.9), (float("nan"), 0.9)):
        assert f(2, a, 0, a, 0, a, a, None, n, (ctypes.c_double * 5)(*bad, 1e-3, 0.1, 1e-8), 1, None, None) == EINVAL
    assert f(2, a, 5, a, 5, a, a, None, n, h, 1, None, None) == EDTYPE
    assert f(2, a, 0, a, 1, a, a, None, n, h, 1, None, None) == EDTYPE        # bf16 gradients of fp32 parameters
    assert f(2, a, 1, a, 2, a, a, None, n, h, 1, None, None) == EDTYPE
    assert f(2, a, 0, a, 0, a, a, a, n, h, 1, None, None) == EDTYPE           # masters of fp32 parameters
    for k in range(4):
        args = [none if j == k else a for j in range(4)]
        assert f(2, args[0], 0, args[1], 0, args[2], args[3], None, n, h, 1, None, None) == EINVAL
        args = [odd if j == k else a for j in range(4)]
        assert f(2, args[0], 0, args[1], 0, args[2], args[3], None, n, h, 1, None, None) == EALIGN
    assert f(2, a, 1, a, 1, a, a, none, n, h, 1, None, None) == EINVAL
    assert f(2, a, 0, a, 0, a, a, None, (i64 * 2)(1, -1), h, 1, None, None) == EINVAL
    assert f(2, a, 0, a, 0, a, a, None, n, h, 1, p + 2, None) == EALIGN
    assert f(1, a, 0, a, 0, a, a, None, (i64 * 1)(1 << 62), h, 1, None, None) == ESHAPE
    assert f(2, none, 0, none, 0, none, none, None, (i64 * 2)(0, 0), h, 1, None, None) == 0
    # memory shared by a tensor that is written: 10 fp32 elements (40 bytes) from each of these
    n10, EOVERLAP = (i64 * 2)(10, 10), -6
    cols = [(vp * 2)(p + 400 * k, p + 400 * k + 200) for k in range(5)]
    assert f(2, a, 0, cols[1], 0, cols[2], cols[3], None, n10, h, 1, None, None) == EOVERLAP                            # a tensor twice
    assert f(2, (vp * 2)(p, p + 36), 0, cols[1], 0, cols[2], cols[3], None, n10, h, 1, None, None) == EOVERLAP          # the last element
    assert f(2, cols[0], 0, cols[0], 0, cols[2], cols[3], None, n10, h, 1, None, None) == EOVERLAP                      # params as grads
    assert f(2, cols[0], 0, (vp * 2)(p + 400, p + 836), 0, cols[2], cols[3], None, n10, h, 1, None, None) == EOVERLAP   # a grad into exp_avg
    assert f(2, cols[0], 1, cols[1], 1, cols[2], cols[3], cols[3], n10, h, 1, None, None) == EOVERLAP                   # a master as a moment
    assert b"shares memory" in L.coat_status_string(EOVERLAP)


def test_binding_is_built_for_this_library_and_refuses_other_objects():
    from coat_amd import _hip
    native = _hip.native()
    assert native is _hip.native() and native.ABI_VERSION == _hip.ABI_VERSION
    t = torch.zeros(4, 8)
    for call in (lambda: native.layer_norm_forward(3, None, None, 1e-5), lambda: native.layer_norm_forward(t, [1.0], None, 1e-5),
                 lambda: native.layer_norm_forward(t, None, None, "eps"), lambda: native.layer_norm_forward(t),
                 lambda: native.grad_norm_multi([t, 3], 1.0), lambda: native.grad_norm_multi(3, 1.0),
                 lambda: native.adamw_step_multi([t], [t], [t], [None], None, 0.9, 0.9, 0.1, 0.1, 1e-8, 1, None),
                 lambda: native.rotary_axes(None, 3, t, t, t, 8, 1, 4, False, False)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        native.bind({}, torch.cuda.current_stream)
    with pytest.raises(RuntimeError, match="GPU"):  # and still holds the library
        native.layer_norm_forward(t, None, None, 1e-5)


def test_python_refusals():
    from coat_amd.activation.norm import layer_norm, layer_norm_forward
    from coat_amd.models.rotary import RotaryAxes, rotary_axes, rotary_axes_forward
    from coat_amd.optimizer import qoptim_cuda

    x = torch.zeros(4, 32)
    for f in (layer_norm, layer_norm_forward):
        with pytest.raises(RuntimeError, match="GPU"):
            f(x)
    for bad in (dict(sections=()), dict(sections=(0, 0)), dict(sections=(-1, 5)), dict(sections=(10, 10)), dict(sections=(4,), theta=0.0),
                dict(sections=(4,), theta=float("inf"))):
        with pytest.raises(ValueError):
            RotaryAxes(32, **bad)
    plan = RotaryAxes(32, (6, 10))
    q, pos = torch.zeros(1, 3, 2, 32), torch.zeros(2, 1, 3, dtype=torch.int64)
    for f in (rotary_axes, rotary_axes_forward):
        with pytest.raises(RuntimeError, match="GPU"):
            f(q, None, pos, plan)
        with pytest.raises(ValueError, match="neither"):
            f(None, None, pos, plan)
    with pytest.raises(RuntimeError, match="GPU"):
        qoptim_cuda.grad_norm_multi([x])
    with pytest.raises(ValueError):
        qoptim_cuda.grad_norm_multi([])
    with pytest.raises(ValueError, match="max_norm"):
        qoptim_cuda.grad_norm_multi([x], max_norm=-1.0)
    with pytest.raises(RuntimeError, match="GPU"):
        qoptim_cuda.adamw_step_multi([x], [x], [x], [x], 0.9, 0.95, 1e-3, 0.1, 1e-8, 1)
    qoptim_cuda.adamw_step_multi([], [], [], [], 0.9, 0.95, 1e-3, 0.1, 1e-8, 1)  # nothing to do


@pytest.mark.gpu
def test_python_refusals_of_gpu_tensors(dev):
    from coat_amd.activation.norm import layer_norm_backward, layer_norm_forward
    from coat_amd.models.rotary import RotaryAxes, rotary_axes_forward
    from coat_amd.optimizer import qoptim_cuda

    x, w = torch.zeros(4, 32, device=dev), torch.ones(32, device=dev)
    stat = torch.ones(4, device=dev)
    for args in ((x.double(),), (x, w[:16]), (x, None, w), (x, w, w.bfloat16()), (x, w.cpu()), (x, w, None, -1.0), (x[:, :0],), (x[0, 0],)):
        with pytest.raises(ValueError):
            layer_norm_forward(*args)
    for args in ((x.bfloat16(), x, stat, stat), (x[:3], x, stat, stat), (x, x, stat[:3], stat), (x, x, stat, stat.double()), (x, x, stat, stat, w[:5])):
        with pytest.raises(ValueError):
            layer_norm_backward(*args)
    plan = RotaryAxes(32, (6, 10))
    q, pos = torch.zeros(1, 3, 2, 32, device=dev), torch.zeros(2, 1, 3, dtype=torch.int64, device=dev)
    for args in ((q[..., :30], None, pos), (q, q.half(), pos), (q, q[:, :2], pos), (q[0], None, pos), (q, None, pos[:1]), (q, None, pos[0]),
                 (q, None, pos.float()), (q, None, pos.cpu()), (q.double(), None, pos)):
        with pytest.raises(ValueError):
            rotary_axes_forward(*args, plan)
    with pytest.raises(RuntimeError):
        rotary_axes_forward(q, None, pos[:, :, :2], plan)  # two positions for three tokens
    a = [torch.zeros(8, device=dev) for _ in range(8)]
    hyper = (0.9, 0.95, 1e-3, 0.1, 1e-8, 1)
    step = qoptim_cuda.adamw_step_multi
    for args in ((a[:2], a[2:3], a[4:6], a[6:]), (a[:2], a[2:4], a[4:6], [a[6], a[7][:4]]), ([a[0], a[0]], a[2:4], a[4:6], a[6:]),
                 (a[:2], a[2:4], a[4:6], a[4:6]), ([a[0], a[1].half()], a[2:4], a[4:6], a[6:]), (a[:2], [a[2], a[3].half()], a[4:6], a[6:]),
                 (a[:2], a[2:4], a[4:6], [a[6], a[7].half()]), (a[:2], [a[2].half(), a[3].half()], a[4:6], a[6:]),
                 (a[:2], [a[2], a[3].cpu()], a[4:6], a[6:])):
        with pytest.raises(RuntimeError):
            step(*args, *hyper)
    flat = torch.zeros(200, 5, 8, device=dev)
    many = [[flat[i, k] for i in range(200)] for k in (0, 1, 2, 3)]
    many[0][150] = many[0][3]  # the same parameter twice, in two launches
    with pytest.raises(RuntimeError, match="twice"):
        step(*many, *hyper)
    assert not flat.any()
    two = torch.zeros(8, 2, device=dev)[:, 0]
    with pytest.raises(RuntimeError, match="contiguous"):
        step([two], [a[1]], [a[2]], [a[3]], *hyper)
    with pytest.raises(ValueError, match="step"):
        step([a[0]], [a[1]], [a[2]], [a[3]], *hyper[:5], 0)
    with pytest.raises(RuntimeError, match="masters"):
        step([a[0]], [a[1]], [a[2]], [a[3]], *hyper, masters=[a[4]])
    for bad in (torch.ones(2, device=dev), torch.ones(1), torch.ones(1, device=dev).double()):
        with pytest.raises(RuntimeError, match="grad_scale"):
            step([a[0]], [a[1]], [a[2]], [a[3]], *hyper, grad_scale=bad)
    assert not any(t.any() for t in a)


def test_scaled_fp8_step_entries(L, p):
    i64, vp = ctypes.c_int64, ctypes.c_void_p
    a, n, s, hp = (vp * 2)(p, p), (i64 * 2)(128, 256), (i64 * 2)(1, 2), (0.9, 0.95, 1e-3, 0.1, 1e-8, 1)
    f, e = L.coat_fp8_adamw_step_multi_scaled, L.coat_fp8_adamw_expand_step_multi_scaled
    assert f(2, a, a, 0, a, a, a, a, n, s, *hp, 128, None, None) == EINVAL  # a factor is what they are for
    assert e(2, a, a, 0, a, a, a, a, a, a, a, a, n, s, *hp, 128, 16, None, None) == EINVAL
    assert f(2, a, a, 0, a, a, a, a, n, s, *hp, 128, p + 2, None) == EALIGN
    assert f(2, a, a, 0, a, a, a, a, n, s, *hp, 64, p, None) == -4
    assert f(2, a, a, 7, a, a, a, a, n, s, *hp, 128, p, None) == EDTYPE
    assert f(0, None, None, 0, None, None, None, None, None, None, *hp, 128, p, None) == 0


def test_optimizer_refusals():
    from coat_amd.optimizer.fp8_adamw import CoatAdamW
    w = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(state_bits=16), dict(master_weights=True), dict(max_grad_norm=-1.0), dict(max_grad_norm=float("nan"))):
        with pytest.raises(ValueError):
            CoatAdamW([w], **bad)
    for bad in (dict(state_bits=4), dict(master_weights=True)):
        with pytest.raises(ValueError):
            CoatAdamW([dict(params=[w], **bad)])
    for kw in (dict(), dict(max_grad_norm=1.0)):  # one norm for all groups
        with pytest.raises(ValueError, match="max_grad_norm"):
            CoatAdamW([dict(params=[w], max_grad_norm=0.5)], **kw)
    again = CoatAdamW([w], max_grad_norm=1.0)
    assert CoatAdamW(again.param_groups, max_grad_norm=1.0).param_groups[0]["max_grad_norm"] == 1.0
    opt = CoatAdamW([w])  # the reference's groups are unchanged where nothing is asked for
    assert set(opt.param_groups[0]) == {"params", "lr", "betas", "eps", "weight_decay", "amsgrad", "fused"}
    assert CoatAdamW([w], state_bits=32, max_grad_norm=0.0).param_groups[0]["state_bits"] == 32
    w.grad = torch.zeros(4)
    for kw in (dict(state_bits=32), dict(max_grad_norm=1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            CoatAdamW([w], **kw).step()


def test_attention_module_evaluates_several_axes_on_the_cpu():
    from coat_amd.models.coat_llama import CoatLlamaConfig, LlamaSdpaAttentionWithoutLinear, apply_rotary_pos_emb
    g = torch.Generator().manual_seed(0)
    config = CoatLlamaConfig(hidden_size=64, num_attention_heads=2, rotary_sections=(4, 6, 6))
    module = LlamaSdpaAttentionWithoutLinear(config).eval()
    q, k, v = (torch.randn(1, 7, 64, generator=g) for _ in range(3))
    pos = torch.randint(0, 50, (3, 1, 7), generator=g)
    out = module(q, k, v, position_ids=pos)[0]
    freq = 10000.0 ** -(torch.arange(16, dtype=torch.float64) / 16)
    ang = torch.cat((pos[0, 0, :, None] * freq[:4], pos[1, 0, :, None] * freq[4:10], pos[2, 0, :, None] * freq[10:]), -1)
    ang = torch.cat((ang, ang), -1)[None]
    heads = [t.view(1, 7, 2, 32).transpose(1, 2).double() for t in (q, k, v)]
    rq, rk = apply_rotary_pos_emb(heads[0], heads[1], ang.cos(), ang.sin())
    s = (rq @ rk.transpose(2, 3) / 32 ** 0.5).masked_fill(torch.triu(torch.ones(7, 7, dtype=torch.bool), 1), float("-inf")).softmax(-1)
    assert torch.allclose(out.double(), (s @ heads[2]).transpose(1, 2).reshape(1, 7, 64), rtol=0, atol=1e-5)
    for bad in (pos[:2], torch.cat((pos, pos))):
        with pytest.raises(ValueError, match="position_ids"):
            module(q, k, v, position_ids=bad)
    with pytest.raises(ValueError, match="rotary_sections"):
        LlamaSdpaAttentionWithoutLinear(CoatLlamaConfig(hidden_size=64, num_attention_heads=2))(q, k, v, position_ids=pos)
