"""Host-side checks of the block operators (nerf_amd/operators.py, nerf_amd/optim.py): no GPU needed.

* what the entry points refuse, in Python and at the C boundary, before anything reaches a device;
* the ctypes structures have the header's layout (compiled from it);
* the 64-bit formulas the GPU tests compare with: their gradients against differences.
"""
import ctypes
import os
import subprocess

import pytest
import torch

import operator_truth as truth
from nerf_amd import operators as ops
from nerf_amd import optim
from nerf_amd import runtime as rt

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------------------------------- layout --
def test_structures_match_header(tmp_path):
    structs = {"nerf_rotary_tensor": rt.RotaryTensor, "nerf_rotary_desc": rt.RotaryDesc, "nerf_block_desc": rt.BlockDesc,
               "nerf_adamw_control": rt.AdamWControl, "nerf_adamw_tensor": rt.AdamWTensor,
               "nerf_adamw_config": rt.AdamWConfig}
    lines = ['#include <stdio.h>', '#include "nerf_mi355x.h"', "int main(void) {"]
    for c, py in structs.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        for name, _ in py._fields_:
            lines.append(f'printf("{c}.{name} %zu\\n", offsetof({c}, {name}));')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    said = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for c, py in structs.items():
        assert int(said[c]) == ctypes.sizeof(py), c
        for name, _ in py._fields_:
            assert int(said[f"{c}.{name}"]) == getattr(py, name).offset, f"{c}.{name}"
    # the one-pack form of the rotary descriptor: every member where ctypes has it
    values = list(range(1, 39))
    d = rt.RotaryDesc.from_buffer_copy(ops._ROTARY.pack(*values))
    assert ops._ROTARY.size == ctypes.sizeof(rt.RotaryDesc)
    got = [d.dtype, d.head_dim, d.n_axes, *d.sections, d.shared_ladder, d.interleaved, d.inverse, int(d.base),
           ctypes.cast(d.frequencies, ctypes.c_void_p).value, d.positions, d.position_dtype, *d.position_stride, d.n_batch,
           d.n_tokens, d.n_tensors]
    for t in d.tensor:
        got += [t.x, t.out, t.heads, *t.x_stride, *t.out_stride]
    assert got == values[:len(got)] and len(got) == len(values)


# ------------------------------------------------------------------------------------------- rotary --
def _rot(**k):
    d = dict(x=torch.zeros(5, 2, 8), positions=torch.zeros(5, 2), sections=(2, 2))
    d.update(k)
    x, p, s = d.pop("x"), d.pop("positions"), d.pop("sections")
    return ops.rotary_axes(x, p, s, **d)


@pytest.mark.parametrize("change, words", [
    (dict(x=torch.zeros(5, 2, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(5, 8)), r"\[tokens, heads, dim\]"),
    (dict(x=torch.zeros(5, 2, 16)[..., ::2]), "contiguous"),
    (dict(x=(torch.zeros(5, 2, 8), torch.zeros(4, 2, 8))), "does not go with"),
    (dict(x=(torch.zeros(5, 2, 8), torch.zeros(5, 2, 8).half())), "does not go with"),
    (dict(x=(torch.zeros(5, 2, 8),) * 3), "one or two"),
    (dict(x=torch.zeros(5, 2, 8, requires_grad=True)), "requires grad"),
    (dict(sections=(3, 2)), "5 pairs"),
    (dict(sections=(5, -1)), "sections"),
    (dict(sections=()), "sections"),
    (dict(sections=(1, 1, 1, 1, 0), positions=torch.zeros(5, 5)), "sections"),
    (dict(positions=torch.zeros(5, 3)), "positions"),
    (dict(positions=torch.zeros(2, 5, 2)), "positions"),
    (dict(positions=torch.zeros(5, 2, dtype=torch.float64)), "positions"),
    (dict(ladder="other"), "ladder"),
    (dict(pairs="other"), "pairs"),
    (dict(frequencies=[1.0]), "4 frequencies"),
    (dict(out=torch.zeros(5, 2, 9)), "out"),
    (dict(out=torch.zeros(1, 1, 8).expand(5, 2, 8)), "repeats"),
    (dict(out=(torch.zeros(5, 2, 8),) * 2), "must be a tensor"),
    (dict(), "device tensors"),
])
def test_rotary_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        _rot(**change)


def test_rotary_refuses_two_outputs_in_one_place():
    x = torch.zeros(5, 2, 8)
    with pytest.raises(ValueError, match="share"):
        _rot(x=(x, x), out=(x, x))
    b = torch.zeros(4, 4, 8)
    with pytest.raises(ValueError, match="another order"):
        ops.rotary_axes(b, torch.zeros(4, 2), (2, 2), out=b.transpose(0, 1))


def _rotary_desc():
    d = rt.RotaryDesc()
    d.dtype, d.head_dim, d.n_axes, d.base = rt.NERF_F32, 8, 1, 10000.0
    d.sections[0] = 4
    d.positions, d.position_dtype = 64, rt.NERF_F32
    d.n_batch, d.n_tokens, d.n_tensors = 1, 2, 1
    t = d.tensor[0]
    t.x, t.out, t.heads = 64, 64, 1
    return d


def _last():
    return rt.load_library().nerf_last_error().decode()


@pytest.mark.parametrize("field, value", [
    ("dtype", 7), ("position_dtype", rt.NERF_FLOAT16), ("n_axes", 0), ("n_axes", 5), ("n_tensors", 0), ("n_tensors", 3),
    ("n_batch", -1), ("n_tokens", -1), ("head_dim", 6), ("base", 0.0), ("base", float("nan")), ("positions", None),
    ("n_tokens", 1 << 50)])
def test_rotary_c_refuses(field, value):
    lib, d = rt.load_library(), _rotary_desc()
    setattr(d, field, value)
    assert lib.nerf_rotary_axes(ctypes.byref(d), None) == -1
    assert "nerf_rotary_axes" in _last()


def test_rotary_c_refuses_tensors():
    lib = rt.load_library()
    assert lib.nerf_rotary_axes(None, None) == -1
    for field, value in (("x", None), ("out", None), ("x", 66), ("heads", -1)):
        d = _rotary_desc()
        setattr(d.tensor[0], field, value)
        assert lib.nerf_rotary_axes(ctypes.byref(d), None) == -1, field
    d = _rotary_desc()
    d.n_tokens = 0        # nothing to do: no launch
    assert lib.nerf_rotary_axes(ctypes.byref(d), None) == 0


# -------------------------------------------------------------------------------------------- block --
def _blk(back=False, **k):
    d = dict(x=torch.zeros(3, 4), w_gate=torch.zeros(6, 4), w_up=torch.zeros(6, 4), w_down=torch.zeros(5, 6))
    dy = k.pop("dy", torch.zeros(3, 5))
    d.update(k)
    args = [d.pop(n) for n in ("x", "w_gate", "w_up", "w_down")]
    return ops.gated_block_backward(dy, *args, **d) if back else ops.gated_block(*args, **d)


@pytest.mark.parametrize("change, words", [
    (dict(x=torch.zeros(3, 4, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(x=torch.zeros(3, 5)), "x must be"),
    (dict(x=torch.zeros(3, 8)[:, ::2]), "contiguous"),
    (dict(x=torch.zeros(1, 4).expand(3, 4)), "overlap"),
    (dict(x=torch.zeros(2, 3, 8)[:, :, :4][:, :2]), "rows of one stride"),
    (dict(w_gate=torch.zeros(6, 4).half()), "w_gate"),
    (dict(w_up=torch.zeros(5, 4)), r"\[hidden, width\]"),
    (dict(w_down=torch.zeros(5, 7)), r"\[out, hidden\]"),
    (dict(w_down=torch.zeros(0, 6)), "w_down"),
    (dict(w_up=torch.zeros(4, 6).t()), "contiguous"),
    (dict(activation="tanh"), "activation"),
    (dict(w_gate=torch.zeros(6, 4, requires_grad=True)), "requires grad"),
    (dict(), "device tensors"),
])
@pytest.mark.parametrize("back", [False, True])
def test_block_refuses(change, words, back):
    with pytest.raises(ValueError, match=words):
        _blk(back, **change)


@pytest.mark.parametrize("change, words", [
    (dict(dy=torch.zeros(3, 6)), "dy"),
    (dict(dy=torch.zeros(2, 5)), "dy"),
    (dict(dy=torch.zeros(3, 5).half()), "dy"),
    (dict(needs=(True, True)), "four"),
    (dict(out=(None, torch.zeros(4, 6).t(), None, None)), "dw_gate"),
    (dict(out=(torch.zeros(2, 4), None, None, None)), "dx"),
])
def test_block_backward_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        _blk(True, **change)


def test_block_out_refusals():
    with pytest.raises(ValueError, match="out must be"):
        _blk(out=torch.zeros(3, 4))
    a = torch.zeros(40)
    with pytest.raises(ValueError, match="overlaps x"):
        ops._refuse_overlap(dict(out=a[4:12]), dict(x=a[:5], w=a[30:]))
    with pytest.raises(ValueError, match="overlaps dx"):
        ops._refuse_overlap(dict(dx=a[4:12], dw=a[8:20]), {})
    ops._refuse_overlap(dict(out=a[4:12]), dict(x=a[:4], w=a[12:]))


def _block_desc():
    d = rt.BlockDesc()
    d.dtype, d.activation, d.rows, d.width, d.hidden, d.out = rt.NERF_F32, 0, 3, 4, 6, 5
    d.x = d.w_gate = d.w_up = d.w_down = 256
    d.ld_x = d.ld_gate = d.ld_up = 4
    d.ld_down = 6
    return d


@pytest.mark.parametrize("field, value", [
    ("dtype", 3), ("activation", 3), ("rows", -1), ("rows", 1 << 40), ("width", 0), ("hidden", 0), ("out", 0), ("width", 1 << 21),
    ("ld_x", 3), ("ld_gate", 3), ("ld_up", 3), ("ld_down", 5), ("x", None), ("w_gate", None), ("w_down", 258)])
def test_block_c_refuses(field, value):
    lib, d = rt.load_library(), _block_desc()
    setattr(d, field, value)
    big = 1 << 30
    assert lib.nerf_gated_block_forward(ctypes.byref(d), 256, 5, 256, big, None) == -1
    assert lib.nerf_gated_block_backward(ctypes.byref(d), 256, 5, 256, 4, 256, 256, 256, 256, big, None) == -1
    assert lib.nerf_gated_block_workspace(ctypes.byref(d), 1) == 0


def test_block_c_refuses_outputs_and_workspaces():
    lib, d = rt.load_library(), _block_desc()
    need = [lib.nerf_gated_block_workspace(ctypes.byref(d), b) for b in (0, 1)]
    assert 0 < need[0] <= need[1]
    f, b, ref = lib.nerf_gated_block_forward, lib.nerf_gated_block_backward, ctypes.byref(d)
    big = 1 << 30
    assert f(ref, None, 5, 256, big, None) == -1
    assert f(ref, 256, 4, 256, big, None) == -1 and f(ref, 258, 5, 256, big, None) == -1
    assert f(ref, 256, 5, 256, need[0] - 1, None) == -1 and f(ref, 256, 5, None, big, None) == -1
    assert f(ref, 256, 5, 128, big, None) == -1
    assert b(ref, None, 5, 256, 4, 256, 256, 256, 256, big, None) == -1
    assert b(ref, 256, 4, 256, 4, 256, 256, 256, 256, big, None) == -1
    assert b(ref, 256, 5, 256, 3, 256, 256, 256, 256, big, None) == -1
    assert b(ref, 256, 5, 256, 4, 257, 256, 256, 256, big, None) == -1
    assert b(ref, 256, 5, 256, 4, 256, 256, 256, 256, need[1] - 1, None) == -1
    assert b(ref, 256, 5, None, 4, None, None, None, None, 0, None) == 0      # nothing asked for
    d.rows = 0
    assert f(ref, None, 5, None, 0, None) == 0


def test_block_workspaces_of_all_types_and_sizes():
    lib, d = rt.load_library(), _block_desc()
    for dtype in (rt.NERF_F32, rt.NERF_BFLOAT16, rt.NERF_FLOAT16):
        for rows in (0, 1, 16, 17, 300, 1 << 20):
            for width, hidden, out in ((1, 1, 1), (64, 128, 64), (1000, 2730, 1001), (4096, 10240, 4096)):
                d.dtype, d.rows, d.width, d.hidden, d.out = dtype, rows, width, hidden, out
                d.ld_x = d.ld_gate = d.ld_up = width
                d.ld_down = hidden
                for back in (0, 1):
                    need = lib.nerf_gated_block_workspace(ctypes.byref(d), back)
                    assert rows == 0 or need > 0 or not back
                    # h, dg and du of every row, padded copies and partials: bounded by the operands' own sizes
                    values = rows * (3 * hidden + width + out + 64) + 8 * (hidden + 64) * (width + out + 64)
                    assert need <= 16 * values + (256 << 20)


# -------------------------------------------------------------------------------------------- adamw --
@pytest.mark.parametrize("k, words", [
    (dict(params=[]), "no parameters"),
    (dict(params=[torch.zeros(0)]), "no values"),
    (dict(params=[torch.zeros(3, dtype=torch.float64)]), "float32, bfloat16 or float16"),
    (dict(params=[torch.zeros(4, 6).t()]), "contiguous"),
    (dict(state_bits=16), "state_bits"),
    (dict(weight_decay=[0.1]), "weight decays"),
    (dict(weight_decay=-1.0), "weight decays"),
    (dict(betas=(0.9, 1.0)), "betas"),
    (dict(eps=-1.0), "eps"),
    (dict(max_norm=0.0), "max_norm"),
    (dict(lr=-1.0), "learning rate"),
    (dict(lr=float("nan")), "learning rate"),
    (dict(), "device tensors"),
])
def test_adamw_refuses(k, words):
    d = dict(params=[torch.zeros(3), torch.zeros(2, 2)])
    d.update(k)
    with pytest.raises(ValueError, match=words):
        optim.AdamW(d.pop("params"), **d)


def test_adamw_refuses_shared_memory():
    a = torch.zeros(10)
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamW([a, a])
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamW([a[:6], a[5:]])


def _adam(bits=32):
    c = rt.AdamWConfig()
    c.lr, c.beta1, c.beta2, c.eps = 1e-3, 0.9, 0.999, 1e-8
    t = (rt.AdamWTensor * 1)()
    t[0].param = t[0].exp_avg = t[0].exp_avg_sq = 256
    t[0].numel = 5
    if bits == 8:
        t[0].exp_avg_scale = t[0].exp_avg_sq_scale = 256
    return c, t


def _plan(t, bits=32):
    lib = rt.load_library()
    plan = (ctypes.c_int64 * (lib.nerf_adamw_plan_bytes(len(t), t, bits) // 8))()
    assert lib.nerf_adamw_plan(len(t), t, bits, plan) == 0
    return plan


@pytest.mark.parametrize("field, value", [
    ("param", 0), ("exp_avg", 0), ("exp_avg_sq", 0), ("numel", -1), ("weight_decay", -1.0), ("weight_decay", float("nan")),
    ("param", 257), ("exp_avg", 254), ("numel", 0), ("numel", 1 << 41)])
def test_adamw_plan_refuses(field, value):
    lib = rt.load_library()
    _, t = _adam()
    setattr(t[0], field, value)
    assert lib.nerf_adamw_plan_bytes(1, t, 32) == 0
    assert lib.nerf_adamw_plan(1, t, 32, (ctypes.c_int64 * 64)()) == -1


def test_adamw_plan_refuses_the_rest():
    lib = rt.load_library()
    _, t = _adam()
    assert lib.nerf_adamw_plan_bytes(1, None, 32) == 0 and lib.nerf_adamw_plan_bytes(0, t, 32) == 0
    assert lib.nerf_adamw_plan_bytes(1, t, 16) == 0
    assert lib.nerf_adamw_plan_bytes(1, t, 8) == 0          # scales missing
    assert lib.nerf_adamw_plan(1, t, 32, None) == -1
    t[0].model, t[0].model_dtype = 256, rt.NERF_F32
    assert lib.nerf_adamw_plan_bytes(1, t, 32) == 0
    assert lib.nerf_adamw_workspace(None) == 0 and lib.nerf_adamw_workspace((ctypes.c_int64 * 8)()) == 0


@pytest.mark.parametrize("field, value", [
    ("lr", -1.0), ("beta1", 1.0), ("beta2", -0.1), ("eps", -1.0), ("flags", 8), ("lr", float("nan")), ("max_norm", float("nan"))])
def test_adamw_c_refuses_settings(field, value):
    lib = rt.load_library()
    c, t = _adam()
    plan = _plan(t)
    g, k = (ctypes.c_uint64 * 1)(256), (ctypes.c_int32 * 1)(0)
    setattr(c, field, value)
    assert lib.nerf_adamw_step(ctypes.byref(c), plan, 256, g, k, 256, None, 0, None) == -1


def test_adamw_c_refuses_the_rest():
    lib = rt.load_library()
    c, t = _adam()
    plan = _plan(t)
    g, k = (ctypes.c_uint64 * 1)(256), (ctypes.c_int32 * 1)(0)
    ok = [ctypes.byref(c), plan, 256, g, k, 256, None, 0, None]
    for at, value in ((0, None), (1, None), (1, (ctypes.c_int64 * 8)()), (2, None), (2, 264), (3, None), (4, None), (5, None),
                      (5, 258), (3, (ctypes.c_uint64 * 1)(258)), (3, (ctypes.c_uint64 * 1)(0)), (4, (ctypes.c_int32 * 1)(3))):
        args = list(ok)
        args[at] = value
        assert lib.nerf_adamw_step(*args) == -1, at
    c.max_norm = 1.0                                 # a norm needs its workspace
    need = lib.nerf_adamw_workspace(plan)
    assert need >= 8
    for ws, size in ((None, need), (256, need - 1), (260, need)):
        assert lib.nerf_adamw_step(*ok[:6], ws, size, None) == -1


def test_trainer_options_are_checked():
    from nerf_amd.trainer import MI355XTrainer

    t = MI355XTrainer.__new__(MI355XTrainer)
    for kind, bits in (("sgd", 32), ("adam", 8), ("adamw", 16)):
        with pytest.raises(ValueError):
            t.set_optimizer(kind, bits)
    import main as cli

    with pytest.raises(SystemExit):
        cli.main(["--optimizer_state_bits", "8"])


# ----------------------------------------------------------------------------------- the formulas --
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
def test_block_truth_against_differences(kind):
    gen = torch.Generator().manual_seed(5)
    x, wg, wu, wd, dy = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((4, 3), (6, 3), (6, 3), (5, 6), (4, 5)))
    got = truth.block(*(v.float() for v in (x, wg, wu, wd)), kind, dy.float())
    x, wg, wu, wd, dy = (v.float().double() for v in (x, wg, wu, wd, dy))

    def loss():
        a, _, _ = truth.act(x @ wg.t(), kind)
        return float((dy * ((a * (x @ wu.t())) @ wd.t())).sum())

    for name, v in (("dx", x), ("dw_gate", wg), ("dw_up", wu), ("dw_down", wd)):
        flat, grad = v.view(-1), got[name][0].reshape(-1)
        for i in range(0, flat.numel(), 5):
            keep, e = float(flat[i]), 1e-6
            flat[i] = keep + e
            hi = loss()
            flat[i] = keep - e
            lo = loss()
            flat[i] = keep
            # central difference: e^2 times a third derivative of a few hundreds, and 1e-15 / e
            assert abs((hi - lo) / (2 * e) - float(grad[i])) < 1e-7, (name, i)


def test_rotary_truth_turns_back():
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(2, 7, 3, 10, generator=gen)
    pos = torch.randint(0, 1000, (2, 7, 2), generator=gen)
    f = truth.ladder((3, 1))
    for inter in (False, True):
        y, _ = truth.rotary(x, pos, (3, 1), f, inter, False)
        z, _ = truth.rotary(y, pos, (3, 1), f, inter, True)
        assert float((z - x.double()).abs().max()) < 1e-12
        assert torch.equal(y[..., 8:], x[..., 8:].double())
        # the turn is orthogonal, so its gradient is the turn back
        assert float((y.norm(dim=-1) - x.double().norm(dim=-1)).abs().max()) < 1e-12


def test_adamw_truth_is_torchs():
    gen = torch.Generator().manual_seed(7)
    p = torch.randn(50, generator=gen, dtype=torch.float64)
    q = torch.nn.Parameter(p.clone())
    opt = torch.optim.AdamW([q], lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.3)
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    for t in range(1, 6):
        g = torch.randn(50, generator=gen, dtype=torch.float64)
        q.grad = g.clone()
        opt.step()
        p, m, v = truth.adamw(p, g, m, v, t, 1e-2, 0.8, 0.95, 1e-6, 0.3)
        assert float((p - q.detach()).abs().max()) < 1e-12
