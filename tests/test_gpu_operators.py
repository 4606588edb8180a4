"""The block operators on the GPU against their formulas in 64 bits (tests/operator_truth.py holds the
formulas and derives every bound)."""
import math

import pytest

torch = pytest.importorskip("torch")

import operator_truth as truth  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------- rotary --
def _rotary_case(dtype, batch, tokens, heads, dim, axes, kind, seed=0):
    gen = _gen(seed)
    x = torch.randn(batch, tokens, heads, dim, generator=gen).to(dtype)
    if kind == "point":
        pos = torch.rand(batch, tokens, axes, generator=gen) * 8 - 4
    else:
        pos = torch.randint(-50, 2_000_000, (batch, tokens, axes), generator=gen)
        pos = pos.int() if kind == "int32" else pos
    return x, pos


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("pairs", ["split", "interleaved"])
@pytest.mark.parametrize("batch, tokens, heads, dim, sections, kind, shared, inverse", [
    (1, 1, 1, 2, (1,), "int64", False, False),              # the smallest call
    (1, 1, 40, 128, (16, 24, 24), "int64", True, False),    # one token
    (2, 37, 3, 64, (8, 12, 12), "int32", False, False),
    (3, 129, 5, 80, (8, 12, 12), "int64", True, True),      # a tail of 16 values
    (1, 300, 4, 32, (5, 5, 5), "point", False, False),      # 15 pairs: no 16-byte halves
    (2, 65, 2, 33, (3, 0, 7, 2), "int64", False, True),     # odd head, an empty axis
    (1, 17, 7, 196, (98,), "point", False, False),
    (1, 5, 2, 512, (100, 156), "int64", True, False),       # most pairs
    (1, 9, 2, 48, (0, 0), "int64", False, False),           # nothing turns: a copy
])
def test_rotary(dtype, pairs, batch, tokens, heads, dim, sections, kind, shared, inverse):
    from nerf_amd.operators import rotary_axes

    x, pos = _rotary_case(dtype, batch, tokens, heads, dim, len(sections), kind, seed=dim)
    want, bound = truth.rotary(x, pos, sections, truth.ladder(sections, shared=shared), pairs == "interleaved", inverse)
    got = rotary_axes(x.cuda(), pos.cuda(), sections, ladder="shared" if shared else "axis", pairs=pairs, inverse=inverse)
    assert got.dtype == dtype
    truth.within(got, want, bound, "turned")
    tail = 2 * sum(sections)
    assert torch.equal(got[..., tail:].cpu(), x[..., tail:])     # bit for bit


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rotary_layouts_in_place_and_queries_with_keys(dtype):
    from nerf_amd.operators import rotary_axes

    gen = _gen(3)
    sections, f = (4, 6, 6), truth.ladder((4, 6, 6))
    qkv = torch.randn(2, 50, 12, 32, generator=gen).to(dtype)     # 8 query, 2 key, 2 value heads in one store
    pos = torch.randint(0, 4000, (50, 3), generator=gen)          # shared by the batch
    dev = qkv.cuda()
    q, k = dev[:, :, :8], dev[:, :, 8:10]
    out = rotary_axes((q, k), pos.cuda(), sections, out=(q, k))
    assert out[0].data_ptr() == q.data_ptr()
    want, bound = truth.rotary(qkv, pos.expand(2, 50, 3), sections, f, False, False)
    truth.within(dev[:, :, :10], want[:, :, :10], bound[:, :, :10], "in place")
    assert torch.equal(dev[:, :, 10:].cpu(), qkv[:, :, 10:])      # the values' heads are as they were
    # heads before tokens: a transposed view in, its strides out; three dimensions; odd strides of an out
    h = qkv.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    got = rotary_axes(h, pos.cuda(), sections)
    assert got.stride() == h.stride()
    truth.within(got, want, bound, "heads first")
    got = rotary_axes(qkv[0].cuda(), pos.cuda(), sections)
    truth.within(got, want[0], bound[0], "three dimensions")
    store = torch.full((2, 50, 12, 37), 7.0, dtype=dtype, device="cuda")
    got = rotary_axes(dev.copy_(qkv), pos.cuda(), sections, out=store[..., 3:35])
    truth.within(got, want, bound, "odd strides")
    assert (store[..., :3] == 7).all() and (store[..., 35:] == 7).all()
    # positions with strides of their own, and a stream of its own
    wide = torch.zeros(50, 3, 5, dtype=torch.int64)
    wide[..., 2] = pos
    side = torch.cuda.Stream()
    x, p = qkv.cuda(), wide.cuda()
    side.wait_stream(torch.cuda.current_stream())
    got = rotary_axes(x, p[..., 2], sections, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    truth.within(got, want, bound, "strided positions on a stream")
    assert rotary_axes(x[:, :0], p[:0, :, 2], sections).shape == (2, 0, 12, 32)


def test_rotary_far_positions_and_frequencies():
    from nerf_amd.operators import rotary_axes

    x = torch.randn(64, 1, 8, generator=_gen(4))
    pos = torch.tensor([[2 ** 40 + 7 * i] for i in range(64)])
    f = [1.0, 0.5, 1e-3, math.pi]
    want, bound = truth.rotary(x, pos, (4,), f, False, False)
    truth.within(rotary_axes(x.cuda(), pos.cuda(), (4,), frequencies=f), want, bound, "far")


def test_rotary_nonfinite_values_stay_in_their_pair():
    from nerf_amd.operators import rotary_axes

    x = torch.ones(1, 2, 12)
    x[0, 0, 3] = float("inf")
    x[0, 1, 11] = float("nan")
    got = rotary_axes(x.cuda(), torch.ones(1, 1, device="cuda"), (4,)).cpu()
    assert not got[0, 0, [3, 7]].isfinite().any() and got[0, 0, [0, 1, 2, 4, 5, 6]].isfinite().all()
    assert got[0, 1, 11].isnan() and got[0, 1, :11].isfinite().all()


# -------------------------------------------------------------------------------------------- block --
def _block_case(dtype, rows, width, hidden, out, seed=0):
    gen = _gen(seed + rows + width)
    x = torch.randn(rows, width, generator=gen).to(dtype)
    wg, wu = ((torch.randn(hidden, width, generator=gen) * width ** -0.5).to(dtype) for _ in "gu")
    wd = (torch.randn(out, hidden, generator=gen) * hidden ** -0.5).to(dtype)
    dy = torch.randn(rows, out, generator=gen).to(dtype)
    return x, wg, wu, wd, dy


def _check_block(case, kind, device_case=None, **k):
    from nerf_amd.operators import gated_block, gated_block_backward

    want = truth.block(*case[:4], kind, case[4])
    x, wg, wu, wd, dy = device_case if device_case is not None else (t.cuda() for t in case)
    truth.within(gated_block(x, wg, wu, wd, activation=kind, **k), *want["y"], "y")
    got = gated_block_backward(dy, x, wg, wu, wd, activation=kind, **k)
    for name, g in zip(("dx", "dw_gate", "dw_up", "dw_down"), got):
        truth.within(g, *want[name], name)


SIZES = [(1, 1, 1, 1), (1, 64, 128, 64), (3, 5, 7, 2), (16, 256, 512, 256), (17, 72, 40, 24), (33, 100, 130, 67),
         (64, 64, 64, 64), (129, 257, 131, 63), (300, 136, 264, 520), (257, 1000, 333, 129), (1000, 31, 65, 33),
         (2, 1536, 700, 300), (700, 512, 512, 512)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows, width, hidden, out", SIZES)
def test_block(dtype, rows, width, hidden, out):
    _check_block(_block_case(dtype, rows, width, hidden, out), "silu")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kind", ["gelu", "relu"])
@pytest.mark.parametrize("rows", [2, 200])
def test_block_activations(dtype, kind, rows):
    _check_block(_block_case(dtype, rows, 96, 160, 96, seed=9), kind)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_block_long_sum_over_rows(dtype):
    # few tiles of weight gradients over many rows
    _check_block(_block_case(dtype, 9001, 40, 56, 24), "silu")


# tall products whose last tiles are cut along k: one of 513 or 514 tiles, and the 129th or 257th of which 128 or 256
# are cut in two, on the larger tile (136 columns) and the smaller
@pytest.mark.parametrize("dtype, rows, width, hidden", [(BF16, 65768, 136, 520), (F16, 65768, 40, 520), (F32, 65768, 136, 520),
                                                        (F32, 32872, 40, 2056), (F32, 32872, 136, 2056)], ids=str)
def test_block_tiles_in_parts(dtype, rows, width, hidden):
    from nerf_amd.operators import gated_block, gated_block_backward

    x, wg, wu, wd, dy = (t.cuda() for t in _block_case(dtype, rows, width, hidden, width))
    want = truth.block(x, wg, wu, wd, "silu", dy)
    truth.within(gated_block(x, wg, wu, wd), *want["y"], "y")
    got = gated_block_backward(dy, x, wg, wu, wd)
    for name, g in zip(("dx", "dw_gate", "dw_up", "dw_down"), got):
        truth.within(g, *want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows, width, hidden, out", [(3001, 100, 300, 60), (9001, 40, 56, 24), (2100, 520, 1300, 520)])
def test_block_any_choice_of_gradients(dtype, rows, width, hidden, out):
    # fewer weight gradients share the machine otherwise, and may need more of the workspace
    from nerf_amd.operators import gated_block_backward

    x, wg, wu, wd, dy = (t.cuda() for t in _block_case(dtype, rows, width, hidden, out))
    want = truth.block(x, wg, wu, wd, "gelu", dy)
    names = ("dx", "dw_gate", "dw_up", "dw_down")
    for mask in range(1, 16):
        needs = tuple(bool(mask >> i & 1) for i in range(4))
        got = gated_block_backward(dy, x, wg, wu, wd, activation="gelu", needs=needs)
        for name, wanted, g in zip(names, needs, got):
            assert (g is not None) == wanted
            if wanted:
                truth.within(g, *want[name], f"{name} of {needs}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 31, 33, 64])
@pytest.mark.parametrize("width, hidden, out", [(2049, 131, 17), (37, 1031, 300), (1000, 4099, 5)])
def test_block_few_rows_of_odd_lengths(dtype, rows, width, hidden, out):
    from nerf_amd.operators import gated_block

    x, wg, wu, wd, _ = _block_case(dtype, rows, width, hidden, out)
    want = truth.block(x, wg, wu, wd, "silu")
    truth.within(gated_block(x.cuda(), wg.cuda(), wu.cuda(), wd.cuda()), *want["y"], "y")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("rows", [60, 64])
def test_block_few_rows_and_wide_weights(dtype, rows):
    # 16-bit weights of 30 MB: the path of few rows ends between these
    from nerf_amd.operators import gated_block

    x, wg, wu, wd, _ = (t.cuda() for t in _block_case(dtype, rows, 1600, 3150, 1560))
    truth.within(gated_block(x, wg, wu, wd), *truth.block(x, wg, wu, wd, "silu")["y"], "y")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows, pad", [(5, 3), (150, 3), (150, 8)])
def test_block_strided_operands(dtype, rows, pad):
    from nerf_amd.operators import gated_block, gated_block_backward

    case = _block_case(dtype, rows, 72, 104, 56, seed=pad)
    dev = []
    for t in case:      # rows inside a wider store, an odd offset in
        store = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=dtype, device="cuda")
        view = store[:, pad // 2:pad // 2 + t.shape[1]]
        view.copy_(t)
        dev.append(view)
    _check_block(case, "silu", dev)
    want = truth.block(*case[:4], "silu", case[4])
    x, wg, wu, wd, dy = dev
    y = torch.full((rows, 56 + pad), 5.0, dtype=dtype, device="cuda")
    gated_block(x, wg, wu, wd, out=y[:, pad - 1:pad - 1 + 56])
    truth.within(y[:, pad - 1:pad - 1 + 56], *want["y"], "strided y")
    assert (y[:, :pad - 1] == 5).all() and (y[:, pad - 1 + 56:] == 5).all()
    dx = torch.full((rows, 72 + pad), 5.0, dtype=dtype, device="cuda")
    got = gated_block_backward(dy, x, wg, wu, wd, needs=(True, False, True, False), out=(dx[:, 1:73], None, None, None))
    assert got[1] is None and got[3] is None
    truth.within(dx[:, 1:73], *want["dx"], "strided dx")
    truth.within(got[2], *want["dw_up"], "dw_up")
    assert (dx[:, :1] == 5).all() and (dx[:, 73:] == 5).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("rows", [3, 140])
def test_block_rows_far_apart(dtype, rows):
    # a tile's rows are 4.7 GB (bf16) and 9.4 GB apart: offsets that pass 32 bits
    from nerf_amd.operators import gated_block, gated_block_backward

    x, wg, wu, wd, dy = (t.cuda() for t in _block_case(dtype, rows, 64, 96, 48))
    step = (1 << 24) + 8
    far = torch.empty(rows * step, dtype=dtype, device="cuda").as_strided((rows, 64), (step, 1))
    far.copy_(x)
    want = truth.block(x, wg, wu, wd, "silu", dy)
    truth.within(gated_block(far, wg, wu, wd), *want["y"], "y")
    for name, g in zip(("dx", "dw_gate", "dw_up", "dw_down"), gated_block_backward(dy, far, wg, wu, wd)):
        truth.within(g, *want[name], name)
    y = torch.empty(rows * step, dtype=dtype, device="cuda").as_strided((rows, 48), (step, 1))
    truth.within(gated_block(x, wg, wu, wd, out=y), *want["y"], "y far apart")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_block_leading_dimensions_and_no_rows(dtype):
    from nerf_amd.operators import gated_block, gated_block_backward

    case = _block_case(dtype, 24, 64, 96, 32)
    x, wg, wu, wd, dy = (t.cuda() for t in case)
    want = truth.block(*case[:4], "silu", case[4])
    y = gated_block(x.view(2, 3, 4, 64), wg, wu, wd)
    assert y.shape == (2, 3, 4, 32)
    truth.within(y.view(24, 32), *want["y"], "y")
    y = gated_block(x[0], wg, wu, wd)
    truth.within(y, want["y"][0][0], want["y"][1][0], "one row")
    dx = gated_block_backward(dy.view(2, 3, 4, 32), x.view(2, 3, 4, 64), wg, wu, wd)[0]
    assert dx.shape == (2, 3, 4, 64)
    truth.within(dx.view(24, 64), *want["dx"], "dx")
    assert gated_block(x[:0], wg, wu, wd).shape == (0, 32)
    none = gated_block_backward(dy[:0], x[:0], wg, wu, wd)
    assert none[0].shape == (0, 64) and all((g == 0).all() for g in none[1:])


def test_block_nonfinite_rows_stay_in_their_row():
    from nerf_amd.operators import gated_block

    for dtype in DTYPES:
        for rows in (4, 200):
            x, wg, wu, wd, _ = _block_case(dtype, rows, 64, 96, 48)
            x[1, 5] = float("inf")
            x[2, 9] = float("nan")
            y = gated_block(x.cuda(), wg.cuda(), wu.cuda(), wd.cuda()).cpu()
            clean = [r for r in range(rows) if r not in (1, 2)]
            assert y[clean].isfinite().all(), dtype
            assert y[2].isnan().all() and not y[1].isfinite().any(), dtype
            want = truth.block(x[clean], wg, wu, wd, "silu")["y"]
            if dtype != F32:        # a 32-bit product's scale may follow the largest finite value: same bound there
                truth.within(y[clean], *want, "clean rows")
            else:
                truth.within(y[clean], *want, "clean rows")


@pytest.mark.parametrize("scale", [1e-12, 1e9])
def test_block_scales_of_32_bits(scale):
    # operands far from 1: 32-bit products must keep their relative accuracy
    from nerf_amd.operators import gated_block, gated_block_backward

    x, wg, wu, wd, dy = _block_case(F32, 130, 64, 96, 48)
    x, wd = x * scale, wd / scale
    want = truth.block(x, wg, wu, wd, "relu", dy)
    x, wg, wu, wd, dy = (t.cuda() for t in (x, wg, wu, wd, dy))
    truth.within(gated_block(x, wg, wu, wd, activation="relu"), *want["y"], "y")
    for name, g in zip(("dx", "dw_gate", "dw_up", "dw_down"), gated_block_backward(dy, x, wg, wu, wd, activation="relu")):
        truth.within(g, *want[name], name)


# fp32 large enough for its operands to be split in halves: odd sizes, values far from 1, columns and rows of their own size
@pytest.mark.parametrize("rows, width, hidden, out, kind, scale", [
    (300, 2301, 1999, 777, "gelu", 1.0), (5000, 333, 1301, 129, "silu", 1.0), (2600, 640, 648, 640, "relu", 1e-12),
    (2600, 640, 648, 640, "relu", 1e9)])
def test_block_halves_of_32_bits(rows, width, hidden, out, kind, scale):
    from nerf_amd.operators import gated_block, gated_block_backward

    x, wg, wu, wd, dy = (t.cuda() for t in _block_case(F32, rows, width, hidden, out))
    x, wd = x * scale, wd / scale
    x[::7] *= 1e-3
    dy[::5] *= 1e4
    wu[3::11] *= 1e-5
    want = truth.block(x, wg, wu, wd, kind, dy)
    truth.within(gated_block(x, wg, wu, wd, activation=kind), *want["y"], "y")
    first = gated_block_backward(dy, x, wg, wu, wd, activation=kind)
    for name, g in zip(("dx", "dw_gate", "dw_up", "dw_down"), first):
        truth.within(g, *want[name], name)
    again = gated_block_backward(dy, x, wg, wu, wd, activation=kind)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_block_halves_nonfinite_rows_and_replays():
    from nerf_amd.operators import gated_block, gated_block_backward

    rows = 1700
    x, wg, wu, wd, dy = (t.cuda() for t in _block_case(F32, rows, 640, 648, 640))
    bad = x.clone()
    bad[1, 5] = float("inf")
    bad[2, 9] = float("nan")
    y = gated_block(bad, wg, wu, wd)
    clean = [r for r in range(rows) if r not in (1, 2)]
    assert y[2].isnan().all() and not y[1].isfinite().any()
    truth.within(y[clean], *truth.block(x[clean], wg, wu, wd, "silu")["y"], "clean rows")
    xin = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gated_block_backward(dy, xin, wg, wu, wd)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (gated_block(xin, wg, wu, wd), *gated_block_backward(dy, xin, wg, wu, wd))
    for i in range(4):
        now = x * (1 + 0.5 * i)
        xin.copy_(now)
        graph.replay()
        want = (gated_block(now, wg, wu, wd), *gated_block_backward(dy, now, wg, wu, wd))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_block_is_deterministic_and_follows_its_stream():
    from nerf_amd.operators import gated_block, gated_block_backward

    for dtype in DTYPES:
        x, wg, wu, wd, dy = (t.cuda() for t in _block_case(dtype, 513, 192, 320, 128))
        first = (gated_block(x, wg, wu, wd), *gated_block_backward(dy, x, wg, wu, wd))
        sides = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in sides:         # two calls at once
            s.wait_stream(torch.cuda.current_stream())
            got.append((gated_block(x, wg, wu, wd, stream=s), *gated_block_backward(dy, x, wg, wu, wd, stream=s)))
        torch.cuda.synchronize()
        for g in got:
            assert all(torch.equal(a, b) for a, b in zip(first, g)), dtype


# -------------------------------------------------------------------------------------------- adamw --
SHAPES = [(1,), (3, 5), (256,), (255, 3), (1024, 4), (77, 129), (0,), (2, 2048), (5000,)]


def _adam_case(dtype, grad_dtype, seed=0, shapes=SHAPES):
    gen = _gen(seed)
    ps = [(torch.randn(*s, generator=gen) * 0.1) for s in shapes]
    gs = [(torch.randn(*s, generator=gen) * 0.01).to(grad_dtype) for s in shapes]
    return ps, [p.to(dtype) for p in ps], gs


def _norm(gs):
    return math.sqrt(sum(float(g.double().square().sum()) for g in gs if g is not None))


@pytest.mark.parametrize("dtype, grad", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)],
                         ids=str)
@pytest.mark.parametrize("max_norm", [None, 0.05])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(dtype, grad, max_norm, bits):
    from nerf_amd.optim import BLOCK, AdamW

    lr, b1, b2, eps = 1e-2, 0.8, 0.95, 1e-6
    full, ps, _ = _adam_case(dtype, grad)
    decay = [0.1 * (i % 3) for i in range(len(ps))]
    dev = [p.cuda() for p in ps]
    opt = AdamW(dev, lr=lr, betas=(b1, b2), eps=eps, weight_decay=decay, state_bits=bits, max_norm=max_norm)
    masters = [p.double() for p in (ps if dtype == F32 else [p.float() for p in ps])]
    for t in range(1, 4):
        gs = _adam_case(dtype, grad, seed=t)[2]
        # each step from the kernel's own last state, so that bounds do not pile up
        m0, v0 = zip(*((m.cpu(), v.cpu()) for m, v in (opt.moments(i) for i in range(len(dev)))))
        p0 = [(p if m is None else m).cpu().reshape(p.shape) for p, m in zip(dev, opt.masters)]
        norm = opt.step([g.cuda() for g in gs])
        factor = 1.0
        if max_norm is not None:
            want = _norm(gs)
            assert abs(float(norm) - want) <= 2.0 ** -23 * want
            factor = min(1.0, max_norm / (want + 1e-6))
            assert factor < 1.0
        else:
            assert norm is None
        for i, g in enumerate(gs):
            p, m, v = truth.adamw(p0[i], g, m0[i], v0[i], t, lr, b1, b2, eps, decay[i], factor)
            size = m0[i].double().abs() + g.double().abs()
            em = 6 * 2.0 ** -24 * size                       # factor, difference, product, sum
            ev = 6 * 2.0 ** -24 * v + 1e-45
            now = (dev[i] if opt.masters[i] is None else opt.masters[i].view(dev[i].shape)).cpu()
            step = lr * (m.abs() + em) / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + eps)
            # p itself rounds twice (decay, sum); the step carries the errors of m and v and eight roundings
            ep = 3 * 2.0 ** -24 * p0[i].double().abs() + step * 20 * 2.0 ** -24 + lr / (1 - b1 ** t) * em / (
                (v / (1 - b2 ** t)).sqrt() + eps)
            truth.within(now, p, ep, f"p {i}")
            if opt.masters[i] is not None:
                assert torch.equal(dev[i].cpu(), now.to(dtype))
            gm, gv = (x.cpu() for x in opt.moments(i))
            if bits == 32:
                truth.within(gm, m, em, f"m {i}")
                truth.within(gv, v, ev, f"v {i}")
            elif g.numel():
                for x, exact, err, root in ((gm, m, em, False), (gv.sqrt(), v.sqrt(), 6 * 2.0 ** -24 * v.sqrt(), True)):
                    n = x.numel()
                    exact, err = exact.reshape(-1), err.reshape(-1)
                    top = torch.nn.functional.pad(exact.abs(), (0, -n % BLOCK)).view(-1, BLOCK).amax(1)
                    scale = (top / 448).repeat_interleave(BLOCK)[:n]
                    # e4m3: half a step is 2^-4 of a normal value and 2^-10 below 2^-6; a root > 0 may
                    # be raised to the smallest code, 2^-9
                    bound = torch.maximum(exact.abs() * 2.0 ** -4, scale * (2.0 ** -9 if root else 2.0 ** -10))
                    truth.within(x.reshape(-1), exact, bound * 1.001 + 2 * err, f"8 bits {i}")
                    if root:
                        assert ((x.reshape(-1) > 0) | (exact == 0)).all()
    assert opt.steps == 3 and opt.skipped == 0


def test_adamw_many_tensors_views_and_missing_gradients():
    from nerf_amd.optim import AdamW

    gen = _gen(11)
    # 150 tensors: four launches; views at odd offsets of one store, 4-byte aligned only
    sizes = [1 + int(x) for x in torch.randint(0, 3000, (150,), generator=gen)]
    starts = [sum(n + 1 for n in sizes[:i]) for i in range(150)]
    store = torch.randn(starts[-1] + sizes[-1] + 5, generator=gen)
    dev = store.cuda()
    params = [dev[s:s + n] for s, n in zip(starts, sizes)]
    opt = AdamW(params, lr=1e-2, weight_decay=0.1, max_norm=1.0)
    grads = [torch.randn(n, generator=gen) if i % 7 else None for i, n in enumerate(sizes)]
    norm = opt.step([None if g is None else g.cuda() for g in grads])
    want = _norm(grads)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    got = dev.cpu()
    touched = torch.zeros_like(store, dtype=torch.bool)
    for i, (s, n, g) in enumerate(zip(starts, sizes, grads)):
        if g is None:
            continue
        touched[s:s + n] = True
        p, m, v = truth.adamw(store[s:s + n], g, torch.zeros(n), torch.zeros(n), 1, 1e-2, 0.9, 0.999, 1e-8, 0.1,
                              min(1.0, 1.0 / (want + 1e-6)))
        truth.within(got[s:s + n], p, 4 * 2.0 ** -24 * store[s:s + n].double().abs() + 1e-2 * 1e-4, f"p {i}")
    assert torch.equal(got[~touched], store[~touched])      # between the tensors and where no gradient was
    with pytest.raises(ValueError, match="no gradients"):
        opt.step([None] * 150)
    with pytest.raises(ValueError, match="gradient 0"):
        opt.step([torch.zeros(sizes[0] + 1, device="cuda")] + [None] * 149)


def test_adamw_skips_what_is_not_finite():
    from nerf_amd.optim import AdamW

    p = [torch.ones(300, device="cuda"), torch.ones(7, device="cuda")]
    opt = AdamW(p, lr=0.1, skip_nonfinite=True, state_bits=8)
    g = [torch.ones(300, device="cuda"), torch.ones(7, device="cuda")]
    opt.step(g)
    kept = [t.clone() for t in p] + [t.view(torch.uint8).clone() for t in opt.exp_avg]
    for bad in (float("inf"), float("nan")):
        g[1][3] = bad
        norm = opt.step(g)
        assert not math.isfinite(float(norm))
        assert all(torch.equal(a, b) for a, b in zip(kept, p + [t.view(torch.uint8) for t in opt.exp_avg]))
    assert opt.steps == 1 and opt.skipped == 2
    g[1][3] = 1.0
    opt.step(g)
    assert opt.steps == 2 and not torch.equal(kept[0], p[0])


def test_adamw_clipped_gradients_and_learning_rates():
    from nerf_amd.optim import AdamW

    p = torch.zeros(1000, device="cuda")
    opt = AdamW([p], lr=torch.tensor([0.5], device="cuda"), max_norm=1.0, write_grads=True, weight_decay=0.0)
    g = torch.full((1000,), 2.0, device="cuda")
    opt.step([g])
    assert abs(float(g.norm()) - 1.0) < 1e-5
    assert torch.allclose(p, torch.full_like(p, -0.5), atol=1e-4)      # the first step is lr * sign
    opt.step([g], lr=0.25)
    assert torch.allclose(p, torch.full_like(p, -0.75), atol=1e-4)
    p2 = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    p2.grad = torch.ones(4, device="cuda")
    AdamW([p2], lr=1.0, weight_decay=0.0).step()
    assert torch.allclose(p2.detach(), torch.full((4,), -1.0, device="cuda"), atol=1e-6)


def test_adamw_refuses_what_shares_memory():
    from nerf_amd.optim import AdamW

    p = [torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")]
    store = torch.zeros(900, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        AdamW(p, state=dict(exp_avg=[store[:300], store[299:599]]))
    with pytest.raises(ValueError, match="share memory"):
        AdamW(p, state=dict(exp_avg=[store[:300], store[300:600]], exp_avg_sq=[store[600:], p[0]]))
    g = torch.ones(300, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        AdamW(p, max_norm=1.0, write_grads=True).step([g, g])
    AdamW(p, max_norm=1.0).step([g, g])       # read only: one gradient of two parameters
    assert torch.equal(p[0], p[1]) and (p[0] != 0).all() and (g == 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_state_round_trip(bits):
    from nerf_amd.optim import AdamW

    def run(opt, n):
        for t in range(n):
            opt.step([g.cuda() for g in _adam_case(BF16, BF16, seed=20 + opt.steps)[2]])

    ps = [p.cuda() for p in _adam_case(BF16, BF16)[1]]
    a = AdamW(ps, lr=1e-2, state_bits=bits, max_norm=0.1)
    run(a, 2)
    qs = [p.clone() for p in ps]
    b = AdamW(qs, lr=1e-2, state_bits=bits, max_norm=0.1)
    state = a.state_dict()
    b.load_state_dict({k: v if k == "steps" else [None if t is None else t.clone() for t in v] for k, v in state.items()})
    run(a, 2)
    run(b, 2)
    assert a.steps == b.steps == 4
    assert all(torch.equal(x, y) for x, y in zip(ps, qs))
    with pytest.raises(ValueError, match="state holds"):
        b.load_state_dict({"steps": 0})


# ------------------------------------------------------------------------------- graphs and the whole --
def test_captured_calls_replay():
    from nerf_amd.operators import gated_block, gated_block_backward, rotary_axes
    from nerf_amd.optim import AdamW

    for dtype in DTYPES:
        x, wg, wu, wd, dy = (t.cuda() for t in _block_case(dtype, 200, 64, 96, 64))
        pos = torch.randint(0, 500, (200, 2), generator=_gen(1)).cuda()

        def step(x, weights, opt):
            turned = rotary_axes(x.view(200, 2, 32), pos, (8, 8)).view(200, 64)
            y = gated_block(turned, *weights)
            d = gated_block_backward(dy, turned, *weights)
            opt.step(d[1:])
            return y, rotary_axes(d[0].view(200, 2, 32), pos, (8, 8), inverse=True)

        eager = [w.clone() for w in (wg, wu, wd)]
        opt_e = AdamW(eager, lr=1e-2, max_norm=1.0)
        mine = [w.clone() for w in (wg, wu, wd)]
        opt_g = AdamW(mine, lr=1e-2, max_norm=1.0)
        warm = [w.clone() for w in (wg, wu, wd)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(x, warm, AdamW(warm, lr=1e-2, max_norm=1.0))
        torch.cuda.current_stream().wait_stream(s)
        xin = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(xin, mine, opt_g)
        for i in range(4):
            now = (x.float() * (1 + 0.1 * i)).to(dtype)
            xin.copy_(now)
            graph.replay()
            want = step(now, eager, opt_e)          # the program's own eager work between the replays
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (dtype, i)
            assert all(torch.equal(a, b) for a, b in zip(mine, eager)), (dtype, i)
        assert opt_g.steps == opt_e.steps == 4


@pytest.mark.parametrize("bits", [32, 8])
def test_a_block_of_point_features_trains(bits):
    """Position-turned point features through a block, its gradients against differences of the loss, and
    a few optimizer steps that run."""
    from nerf_amd.operators import gated_block, gated_block_backward, rotary_axes
    from nerf_amd.optim import AdamW

    gen = _gen(40)
    n, heads, dim, hidden, out = 96, 2, 12, 40, 3
    width = heads * dim
    feats = torch.randn(n, heads, dim, generator=gen).cuda()
    points = (torch.rand(n, 3, generator=gen) * 4 - 2).cuda()
    target = torch.rand(n, out, generator=gen).cuda()
    ws = [(torch.randn(*s, generator=gen) * s[1] ** -0.5).cuda() for s in ((hidden, width), (hidden, width), (out, hidden))]
    freqs = [2.0 ** j * math.pi for j in range(2)] * 3

    def forward(f):
        t = rotary_axes(f, points, (2, 2, 2), frequencies=freqs)
        return t, gated_block(t.view(n, width), *ws)

    def loss64(f, w):
        t, _ = truth.rotary(f.cpu(), points.cpu(), (2, 2, 2), freqs, False, False)
        x, (g, u, d) = t.view(n, width), (v.double().cpu() for v in w)
        a, _, _ = truth.act(x @ g.t(), "silu")
        return float(((a * (x @ u.t())) @ d.t() - target.double().cpu()).square().mean())

    t, y = forward(feats)
    dy = 2 * (y - target) / y.numel()
    grads = gated_block_backward(dy, t.view(n, width), *ws)
    dfeats = rotary_axes(grads[0].view(n, heads, dim), points, (2, 2, 2), frequencies=freqs, inverse=True)
    # directional derivatives: the fp32 gradients are good to ~1e-5 of their size, a central difference
    # in 64 bits to e^2 times a third derivative
    for name, v, g in (("features", feats, dfeats), ("gate", ws[0], grads[1]), ("up", ws[1], grads[2]), ("down", ws[2], grads[3])):
        way = torch.randn(*v.shape, generator=gen).cuda()
        e = 1e-4
        ends = []
        for sign in (1, -1):
            moved = v.double() + sign * e * way.double()
            ends.append(loss64(moved if name == "features" else feats.double(),
                               [moved if v is w else w for w in ws]))
        want = (ends[0] - ends[1]) / (2 * e)
        size = float((g.double().abs() * way.double().abs()).sum())
        assert abs(float((g.double() * way.double()).sum()) - want) <= 2e-5 * size + 1e-6, name
    opt = AdamW(ws, lr=1e-2, max_norm=1.0, state_bits=bits, weight_decay=0.0)
    for _ in range(5):
        t, y = forward(feats)
        dy = 2 * (y - target) / y.numel()
        opt.step(gated_block_backward(dy, t.view(n, width), *ws, needs=(False, True, True, True))[1:])
    assert opt.steps == 5 and all(w.isfinite().all() for w in ws)


# ------------------------------------------------------------------------------------ the trainer --
def _trainer(**config):
    from nerf_amd import weights as W
    from nerf_amd.trainer import MAIN_CONFIG, MI355XTrainer

    sd = W.synthetic_models(0)
    return MI355XTrainer(dict(MAIN_CONFIG, n_rays=64, n_coarse=16, n_fine=32, weight_decay=0.1, **config), *sd)


def _batch(gen):
    pose = torch.eye(4)
    pose[2, 3] = 4.0
    return {"image": torch.rand(16, 16, 3, generator=gen), "pose": pose, "focal": 20.0}


def test_trainer_adamw_is_torchs_step():
    import numpy as np

    tr = _trainer(optimizer="adamw")
    gen = _gen(50)
    batch = _batch(gen)
    params = [torch.nn.Parameter(torch.from_numpy(v.copy()).double()) for sd in tr.state_dicts() for v in sd.values()]
    opt = torch.optim.AdamW(params, lr=3e-4, weight_decay=0.1)
    for t in range(3):
        sel = torch.randperm(256, generator=gen)[:64]
        lr = tr.lr
        tr.train_step(batch, sel, torch.rand(64, 16, generator=gen))
        for q, g in zip(params, [g for net in (0, 1) for g in tr.grads(net).values()]):
            q.grad = torch.from_numpy(g.copy()).double()       # clipped, as param.grad is after the step
        opt.param_groups[0]["lr"] = lr
        opt.step()
        # the trainer's lr decays by lr_gamma; parameters to 3 roundings and 1e-5 of a step each time
        for q, v in zip(params, [v for sd in tr.state_dicts() for v in sd.values()]):
            assert np.abs(q.detach().numpy() - v).max() <= (t + 1) * (3 * 2.0 ** -24 * np.abs(v).max() + 1e-5 * 3e-4 * 10)
    assert tr.steps == 3


def test_trainer_adamw_8_bits_reads_writes_and_resumes(tmp_path):
    import numpy as np

    tr = _trainer(optimizer="adamw", optimizer_state_bits=8)
    gen = _gen(51)
    batch = _batch(gen)
    draws = [(torch.randperm(256, generator=gen)[:64], torch.rand(64, 16, generator=gen)) for _ in range(4)]
    for d in draws[:2]:
        tr.train_step(batch, *d)
    path = tr.save_checkpoint(str(tmp_path / "c.pth"))
    again = _trainer(optimizer="adamw", optimizer_state_bits=8)
    again.load_checkpoint(path)
    assert again.steps == 2
    for net in (0, 1):
        for f in ("exp_avg", "exp_avg_sq"):
            for k, v in getattr(tr, f)(net).items():
                # codes survive; the scale is formed anew from the largest value: two roundings
                assert np.allclose(getattr(again, f)(net)[k], v, rtol=1e-6, atol=0.0), k
    plain = _trainer(optimizer="adamw")
    plain.load_checkpoint(path)
    before = plain.exp_avg_sq(1)
    plain.set_optimizer("adamw", 8)            # fp32 moments become 8-bit ones ...
    for k, v in plain.exp_avg_sq(1).items():
        assert np.allclose(np.sqrt(v), np.sqrt(before[k]), rtol=2.0 ** -4 * 1.01, atol=2.0 ** -9 * np.sqrt(before[k].max()) / 448)
    plain.set_optimizer("adamw", 32)           # ... and stay what they are
    plain.set_optimizer("adam", 32)
    for t in (tr, again):
        for d in draws[2:]:
            t.train_step(batch, *d)
    for a, b in zip(tr.state_dicts(), again.state_dicts()):
        for k in a:
            # two steps apart by the scales' last bits
            assert np.abs(a[k] - b[k]).max() <= 1e-5, k
    with pytest.raises(ValueError):
        tr.set_optimizer("adam", 8)
