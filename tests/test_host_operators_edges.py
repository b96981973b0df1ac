"""CPU: calls of LayerNorm, multi-axis rotary, gradient norm and 32-bit AdamW at the edges of what they promise."""
import pytest
import torch

HYPER = (0.9, 0.95, 1e-3, 0.1, 1e-8, 1)


def binding_calls(x):
    """Every entry of the binding that computes, on ``x`` [4, 8]; on the CPU each ends in a refusal."""
    from coat_amd import _hip
    native, stat, w = _hip.native(), torch.zeros(4), torch.zeros(8)
    turns, axis = torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int32)
    return {"forward": lambda: native.layer_norm_forward(x, None, None, 1e-5),
            "backward": lambda: native.layer_norm_backward(x, x, stat, stat, w, True, True, True),
            "rotary": lambda: native.rotary_axes(x.view(1, 4, 1, 8), None, torch.zeros(1, 1, 4, dtype=torch.int64), turns, axis, 8, 1, 4, False, False, 0),
            "norm": lambda: native.grad_norm_multi([stat, x], 1.0),
            "step": lambda: native.adamw_step_multi([stat, x], [stat, x], [stat, x], [stat, x], None, *HYPER, None)}


# ------------------------------------------------------------------------------------------------ what torch cannot see
@pytest.mark.parametrize("which", ["forward", "backward", "rotary", "norm", "step"])
def test_forward_mode_tangents_are_refused_and_not_lost(which):
    import torch.autograd.forward_ad as fwAD
    x = torch.randn(4, 8)
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            binding_calls(fwAD.make_dual(x, torch.ones_like(x)))[which]()
        with pytest.raises(RuntimeError, match="GPU"):  # a tensor without a tangent is none of this
            binding_calls(x)[which]()


def test_autograd_wrappers_refuse_tangents_with_and_without_requires_grad():
    import torch.autograd.forward_ad as fwAD

    from coat_amd.activation.norm import layer_norm
    from coat_amd.models.rotary import RotaryAxes, rotary_axes
    plan, pos = RotaryAxes(8, (2, 2)), torch.zeros(2, 1, 4, dtype=torch.int64)
    x = torch.randn(1, 4, 1, 8)
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError):
            layer_norm(fwAD.make_dual(x, x))
        with pytest.raises(NotImplementedError):
            rotary_axes(fwAD.make_dual(x, x), None, pos, plan)


@pytest.mark.parametrize("which", ["forward", "backward", "rotary", "norm", "step"])
def test_recordings_of_operations_refuse_the_bare_calls(which):
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(4, 8)

    def f(x):
        binding_calls(x)[which]()
        return x

    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(f, (x,))
    with pytest.raises(NotImplementedError, match="trace"):
        make_fx(f)(x)


@pytest.mark.parametrize("grad", [False, True])
def test_a_trace_records_the_wrappers_as_one_step(grad, monkeypatch):
    """The binding replaced by numpy on the CPU: what the traced function returns for other inputs."""
    from coat_amd import _hip
    from coat_amd.activation.norm import layer_norm
    from coat_amd.models.rotary import RotaryAxes, rotary_axes

    class Native:
        @staticmethod
        def layer_norm_forward(x, w, b, eps):
            y = torch.empty_like(x)
            y.detach().numpy()[...] = x.detach().numpy() * 2
            return y, torch.empty(x.shape[:-1]), torch.empty(x.shape[:-1])

        @staticmethod
        def rotary_axes(q, k, *rest):
            out = torch.empty_like(q)
            out.detach().numpy()[...] = q.detach().numpy() + 1
            return out, None

    monkeypatch.setattr(_hip, "native", lambda: Native)
    plan, pos = RotaryAxes(8, (2, 2)), torch.zeros(2, 1, 4, dtype=torch.int64)
    a, b = (torch.randn(1, 4, 1, 8).requires_grad_(grad) for _ in range(2))
    with pytest.warns(torch.jit.TracerWarning):  # numpy in the stand-in
        norm = torch.jit.trace(lambda x: layer_norm(x), (a,), check_trace=False)
        turn = torch.jit.trace(lambda x: rotary_axes(x, None, pos, plan)[0], (a,), check_trace=False)
    assert torch.equal(norm(b), b * 2) and torch.equal(turn(b), b + 1)


# ------------------------------------------------------------------------------------------------ rotary plans
def test_plans_are_saved_and_copied_without_their_tables():
    """Tables of another device under the key of the first one would be read as that device's memory."""
    import copy
    import io

    from coat_amd.models.rotary import RotaryAxes
    plan, there = RotaryAxes(32, (6, 10), theta=500.0, restart=True, pairs=True), torch.device("cuda", 0)
    old = {**plan.__dict__, "_tables": {there: (torch.zeros(16, dtype=torch.float64), torch.zeros(16, dtype=torch.int32))}}
    plan._tables.update(old["_tables"])
    buffer = io.BytesIO()
    torch.save(plan, buffer)
    buffer.seek(0)
    loaded, before = torch.load(buffer, map_location="cpu", weights_only=False), RotaryAxes.__new__(RotaryAxes)
    before.__setstate__(old)  # a file that still holds tables
    for other in (loaded, before, copy.copy(plan), copy.deepcopy(plan)):
        assert there not in other._tables or other._tables[there][0].device == there
        assert {k: v for k, v in other.__dict__.items() if k not in ("_tables", "_home")} == {k: v for k, v in plan.__dict__.items() if k not in ("_tables", "_home")}
        turns, axis = other.tables(torch.device("cpu"))
        assert turns.tolist() == plan.tables(torch.device("cpu"))[0].tolist() and axis.tolist() == [0] * 6 + [1] * 10


def test_tables_that_are_not_a_plans_are_refused():
    from coat_amd import _hip
    q, pos = torch.zeros(1, 3, 2, 8), torch.zeros(2, 1, 3, dtype=torch.int64)
    turns, axis = torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int32)
    for bad in ((turns.float(), axis), (turns, axis.long()), (turns[:3], axis), (turns, axis[:3]), (torch.zeros(8, dtype=torch.float64)[::2], axis),
                (turns, torch.zeros(8, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError, match="tables"):
            _hip.native().rotary_axes(q, None, pos, *bad, 8, 2, 4, False, False, 0)


def test_plans_keep_no_tables_of_tensors_without_memory():
    """Tables made while a model runs on fake tensors would be refused by every later call."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from coat_amd.models.rotary import RotaryAxes
    plan, cpu = RotaryAxes(32, (6, 10)), torch.device("cpu")
    with FakeTensorMode():
        assert plan.tables(cpu)[0].shape == (16,)
    turns, axis = plan.tables(cpu)
    assert type(turns) is type(axis) is torch.Tensor and turns[0].item() > 0.1


def test_tables_appear_after_their_stream():
    """A thread that finds the tables of another one's first call must find the stream they belong to."""
    from coat_amd.models.rotary import RotaryAxes

    class Order(dict):
        def __setitem__(self, key, value):
            assert key in plan._home
            super().__setitem__(key, value)

    plan = RotaryAxes(32, (6, 10))
    plan._tables = Order()
    plan.tables(torch.device("cpu"))


# ------------------------------------------------------------------------------------------------ CoatAdamW
class Calls:
    """The kernels' Python entries replaced: what the optimizer hands them."""

    def __init__(self, monkeypatch):
        from coat_amd.optimizer import qoptim_cuda
        self.clip, self.steps = [], []
        monkeypatch.setattr(qoptim_cuda, "grad_norm_multi", lambda grads, most: self.clip.append(most) or (torch.tensor(2.0), torch.tensor(0.25)))
        for name in ("adamw_step_multi", "fp8_adamw_expand_step_multi", "fp8_adamw_step_multi", "fp8_adamw_expand_step", "fp8_adamw_step"):
            monkeypatch.setattr(qoptim_cuda, name, lambda *a, _name=name, **kw: self.steps.append((_name, a, kw)))


def parameter(n=4):
    p = torch.nn.Parameter(torch.zeros(n))
    p.grad = torch.ones(n)
    return p


def test_clipping_follows_the_parameter_groups(monkeypatch):
    from coat_amd.optimizer.fp8_adamw import CoatAdamW
    calls = Calls(monkeypatch)
    first = CoatAdamW([parameter()], state_bits=32, max_grad_norm=0.5)
    first.step()
    assert calls.clip == [0.5] and first.grad_norm == 2.0
    for kw in (dict(), dict(state_bits=32), dict(max_grad_norm=3.0)):
        resumed = CoatAdamW([parameter()], **kw)
        resumed.load_state_dict(first.state_dict())
        assert resumed.param_groups[0]["max_grad_norm"] == 0.5
        resumed.step()
        assert calls.clip.pop() == 0.5 and calls.steps[-1][2]["grad_scale"] == 0.25
    first.param_groups[0]["max_grad_norm"] = 0.01
    first.step()
    assert calls.clip[-1] == 0.01
    first.add_param_group(dict(params=[parameter()]))  # joins the others
    assert first.param_groups[1]["max_grad_norm"] == 0.01
    with pytest.raises(ValueError, match="max_grad_norm"):
        first.add_param_group(dict(params=[parameter()], max_grad_norm=0.5))
    first.step()
    for group in first.param_groups:
        group["max_grad_norm"] = None
    n = len(calls.clip)
    first.step()
    assert len(calls.clip) == n and calls.steps[-1][2]["grad_scale"] is None
    first.add_param_group(dict(params=[parameter()]))
    first.step()
    assert len(calls.clip) == n
    first.param_groups[1]["max_grad_norm"] = 1.0
    steps, counts = len(calls.steps), [int(s["step"]) for s in first.state.values()]
    with pytest.raises(ValueError, match="max_grad_norm"):
        first.step()
    assert len(calls.steps) == steps and [int(s["step"]) for s in first.state.values()] == counts  # before anything is stepped


def test_states_that_say_nothing_of_bits_masters_and_clipping_keep_the_optimizers(monkeypatch):
    from coat_amd.optimizer.fp8_adamw import CoatAdamW
    calls, mine = Calls(monkeypatch), dict(state_bits=32, master_weights=True, max_grad_norm=0.5)
    half = torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16))
    opt = CoatAdamW([half], **mine)
    opt.load_state_dict(CoatAdamW([parameter()]).state_dict())  # nothing stepped yet: no moments that could not fit
    assert all(opt.param_groups[0][k] == v for k, v in mine.items())
    half.grad = torch.ones_like(half)
    opt.step()
    name, args, kw = calls.steps[-1]
    assert name == "adamw_step_multi" and kw["masters"][0].dtype == torch.float32 and calls.clip == [0.5]
    p = parameter()
    other = torch.optim.AdamW([p], lr=0.02)
    other.step()
    opt = CoatAdamW([p], **mine)
    opt.load_state_dict(other.state_dict())  # fp32 moments of torch's AdamW
    assert opt.param_groups[0]["lr"] == 0.02 and opt.param_groups[0]["state_bits"] == 32
    opt.step()
    assert calls.steps[-1][0] == "adamw_step_multi" and calls.steps[-1][1][2][0] is opt.state[p]["exp_avg"] and int(opt.state[p]["step"]) == 2
    eight = CoatAdamW([parameter()])
    eight.step()
    opt = CoatAdamW([parameter()], state_bits=32)
    with pytest.raises(ValueError, match="state_bits=32"):
        opt.load_state_dict(eight.state_dict())
    assert not opt.state and opt.param_groups[0]["state_bits"] == 32  # nothing taken over
    opt = CoatAdamW([dict(params=[parameter()], state_bits=8)], state_bits=32)  # a group of its own
    opt.load_state_dict(eight.state_dict())
    opt.step()
    assert opt.param_groups[0]["state_bits"] == 8 and calls.steps[-1][0] in ("fp8_adamw_expand_step", "fp8_adamw_step")
    opt = CoatAdamW([parameter()], state_bits=32, master_weights=True)
    with pytest.raises(ValueError, match="master_weights"):
        opt.load_state_dict(CoatAdamW([dict(params=[parameter()], state_bits=8)], state_bits=32).state_dict())
    restored = CoatAdamW([parameter()])  # and what the state does say is restored, as before
    wide = CoatAdamW([parameter()], state_bits=32)
    wide.step()
    restored.load_state_dict(wide.state_dict())
    assert restored.param_groups[0]["state_bits"] == 32
    restored.step()
    assert calls.steps[-1][0] == "adamw_step_multi"


def test_the_norm_is_that_of_the_last_step(monkeypatch):
    from coat_amd.optimizer.fp8_adamw import CoatAdamW
    Calls(monkeypatch)
    p = parameter()
    opt = CoatAdamW([p], state_bits=32, max_grad_norm=0.5)
    opt.step()
    assert opt.grad_norm == 2.0
    p.grad = None
    opt.step()
    assert opt.grad_norm is None


# ------------------------------------------------------------------------------------------------ sizes of launches
STEP_BLOCKS, STEP_CHUNK, STEP_TENSORS = (2 ** 32 - 1) // 256, 1024, 76


@pytest.fixture(scope="module")
def runs(tmp_path_factory):
    """The library's own split of a list into launches, compiled for the host alone: [(first, last, chunks)] and the status."""
    import ctypes
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "coat_amd", "csrc")
    where = tmp_path_factory.mktemp("runs")
    (where / "runs.cpp").write_text(f'#include "{csrc}/tensor_list.h"\n' + """
extern "C" int64_t max_blocks(int threads) { return coat_max_blocks(threads); }
extern "C" int runs(int count, const int64_t* numel, int64_t chunk, int most, int64_t most_chunks, int64_t* out, int* n) {
    *n = 0;
    return coat_for_each_launch(count, numel, chunk, most, most_chunks, [&](int first, int last, int64_t chunks) {
        int64_t* o = out + 3 * (*n)++;
        o[0] = first, o[1] = last, o[2] = chunks;
        return COAT_OK;
    });
}""")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-o", str(where / "runs.so"), str(where / "runs.cpp")], check=True)
    lib = ctypes.CDLL(str(where / "runs.so"))
    lib.max_blocks.restype = ctypes.c_int64

    def f(numel, chunk=STEP_CHUNK, most=STEP_TENSORS, most_chunks=STEP_BLOCKS):
        assert lib.max_blocks(256) == STEP_BLOCKS
        out, n = (ctypes.c_int64 * (3 * len(numel) + 3))(), ctypes.c_int()
        status = lib.runs(len(numel), (ctypes.c_int64 * len(numel))(*numel), ctypes.c_int64(chunk), most, ctypes.c_int64(most_chunks), out, ctypes.byref(n))
        return status, [tuple(out[3 * i:3 * i + 3]) for i in range(n.value)]

    return f


def test_lists_are_split_into_launches_that_can_start(runs):
    """HIP takes fewer than 2^32 threads: 2^24 - 1 blocks of 256."""
    for numel in ([2 ** 33] * 5, [2 ** 34 - 1024, 1024, 2 ** 34 - 1024], [1, 2 ** 34 - 1024, 0, 1, 0], [5] * 200, [0] * 10, [], [2 ** 28 + 1] * 150,
                  [0, 0, 2 ** 34 - 2048, 1, 1024, 0]):
        status, launches = runs(numel)
        assert status == 0
        covered = [i for first, last, _ in launches for i in range(first, last) if numel[i]]
        assert covered == [i for i, n in enumerate(numel) if n]  # each tensor once, in order
        for first, last, chunks in launches:
            assert chunks == sum(-(-n // STEP_CHUNK) for n in numel[first:last]) and chunks * 256 < 2 ** 32
            assert 1 <= sum(n > 0 for n in numel[first:last]) <= STEP_TENSORS
    assert runs([2 ** 34 - 1023])[0] == runs([4, 2 ** 34])[0] == -2  # COAT_ESHAPE


def test_steps_of_tensors_that_no_launch_takes_are_refused_before_the_first():
    import ctypes

    from coat_amd import _hip
    L, p = _hip.lib(), 1 << 12
    vp, hyper = ctypes.c_void_p * 2, (ctypes.c_double * 5)(0.9, 0.95, 1e-3, 0.1, 1e-8)
    cols = [vp(p + (k << 50), p + (k << 50) + (1 << 48)) for k in range(1, 5)]
    for n in (2 ** 34 - 1023, 2 ** 34, 2 ** 40):
        assert L.coat_adamw_step_multi(2, cols[0], 1, cols[1], 1, cols[2], cols[3], None, (ctypes.c_int64 * 2)(8, n), hyper, 1, None, None) == -2


@pytest.mark.parametrize("count", [77, 153, 200])
def test_shared_memory_is_found_over_all_launches_of_a_step(count):
    """Each pair below lies in two launches; nothing is launched."""
    import ctypes

    from coat_amd import _hip
    L, vp, base = _hip.lib(), ctypes.c_void_p * count, 1 << 40
    numel, hyper = (ctypes.c_int64 * count)(*[100] * count), (ctypes.c_double * 5)(0.9, 0.95, 1e-3, 0.1, 1e-8)
    cols = [[base + (k << 30) + 400 * i for i in range(count)] for k in range(5)]  # 100 fp32 elements from each

    def status(change, p_dtype=0, masters=False):
        c = [list(col) for col in cols]
        for (col, i), at in change.items():
            c[col][i] = at
        a = [vp(*col) for col in c]
        return L.coat_adamw_step_multi(count, a[0], p_dtype, a[1], p_dtype, a[2], a[3], a[4] if masters else None, numel, hyper, 1, None, None)

    last = count - 1
    assert status({(0, last): cols[0][0]}) == -6                                # a parameter twice
    assert status({(0, last): cols[0][0] + 396}) == -6                          # its last element
    assert status({(1, last): cols[0][0] + 4}) == -6                            # a gradient inside an earlier parameter
    assert status({(1, 0): cols[3][last]}) == -6                                # a later moment
    assert status({(2, last): cols[3][0] - 396}) == -6                          # a moment into another one
    assert status({(4, last): cols[2][0] + 200}, p_dtype=1, masters=True) == -6  # a master into a moment


def test_rows_that_are_not_held_in_registers_need_their_workspace():
    import ctypes
    import os
    import re

    from coat_amd import _hip
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    longest = int(re.search(r"#define COAT_LAYER_NORM_ROW (\d+)", open(os.path.join(root, "include", "coat_hip.h")).read()).group(1))
    keep = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(keep) + 15) & ~15
    L = _hip.lib()
    assert L.coat_layer_norm_partials(1, longest) == L.coat_layer_norm_partials(1, longest + 1) == 1
    assert L.coat_layer_norm_backward(p, 0, p, 0, 0, p, p, p, 0, p, p, p, None, 1, 1, longest + 1, None) == -1


# ------------------------------------------------------------------------------------------------ the decoder layer
def test_attention_on_the_cpu_turns_a_part_of_the_head_as_the_gpu_does():
    from coat_amd.models.coat_llama import CoatLlamaConfig, LlamaSdpaAttentionWithoutLinear, apply_rotary_pos_emb
    g = torch.Generator().manual_seed(0)
    config = CoatLlamaConfig(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, rotary_sections=(3, 2, 6))  # 22 of 32 elements
    module = LlamaSdpaAttentionWithoutLinear(config).eval()
    q, k, v = (torch.randn(1, 7, n, generator=g) for n in (64, 32, 32))
    pos = torch.randint(0, 50, (3, 1, 7), generator=g)
    out = module(q, k, v, position_ids=pos)[0]
    freq = 10000.0 ** -(torch.arange(11, dtype=torch.float64) / 11)
    ang = torch.cat((pos[0, 0, :, None] * freq[:3], pos[1, 0, :, None] * freq[3:5], pos[2, 0, :, None] * freq[5:]), -1)
    ang = torch.cat((ang, ang), -1)[None]
    heads = [t.view(1, 7, -1, 32).transpose(1, 2).double().expand(1, 2, 7, 32) for t in (q, k, v)]
    turned = apply_rotary_pos_emb(heads[0][..., :22], heads[1][..., :22], ang.cos(), ang.sin())
    rq, rk = (torch.cat((t, h[..., 22:]), -1) for t, h in zip(turned, heads))
    s = (rq @ rk.transpose(2, 3) / 32 ** 0.5).masked_fill(torch.triu(torch.ones(7, 7, dtype=torch.bool), 1), float("-inf")).softmax(-1)
    assert torch.allclose(out.double(), (s @ heads[2]).transpose(1, 2).reshape(1, 7, 64), rtol=0, atol=1e-5)
