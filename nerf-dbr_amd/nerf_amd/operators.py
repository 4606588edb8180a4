"""Block operators on the MI355X: rotary positions with several axes and the gated feed-forward block.

They stand beside ``runtime.positional_encoding`` and ``Device.query``: torch device tensors in and
out, one call into the HIP library each (``nerf_rotary_axes``, ``nerf_gated_block_forward``,
``nerf_gated_block_backward`` in include/nerf_mi355x.h), queued on torch's current stream of the
tensors' device or on ``stream``.  Nothing is computed in PyTorch and nothing is recorded by
autograd: the gradients are calls of their own (``inverse=True`` for the rotation,
``gated_block_backward`` for the block), and a tensor that requires grad while grad mode is on is
refused.  Workspaces are allocated per call on the call's stream, so a call can be captured into a
graph and two captured graphs share nothing.

The reference has no counterpart: its networks are ReLU chains on sin / cos encodings
(``src/models/nerf.py``).
"""
from __future__ import annotations

import ctypes
from contextlib import ExitStack
from typing import Optional, Sequence

from . import runtime as rt

PAIRS = ("split", "interleaved")
LADDERS = ("axis", "shared")
ACTIVATIONS = {"silu": rt.NERF_SILU, "gelu": rt.NERF_GELU, "relu": rt.NERF_RELU}


def _dtypes():
    import torch

    return {torch.float32: rt.NERF_F32, torch.bfloat16: rt.NERF_BFLOAT16, torch.float16: rt.NERF_FLOAT16}


def _check_plain(torch, **tensors) -> None:
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires grad: the operators are not recorded by autograd (detach it or use "
                             "torch.no_grad(); the gradients are calls of their own)")


class _On(ExitStack):
    """The device and stream a call runs on: current while tensors are allocated and work is queued."""

    def __init__(self, torch, device, stream, **tensors):
        super().__init__()
        for name, t in tensors.items():
            if t.device != device:
                raise ValueError(f"{name} is on {t.device}, not on {device}")
        if device.type != "cuda":
            raise ValueError(f"device tensors are needed, got {device}")
        if stream is not None and stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, not on {device}")
        if torch.cuda.current_device() != device.index:
            self.enter_context(torch.cuda.device(device))
        if stream is not None:
            self.enter_context(torch.cuda.stream(stream))
        self.stream = int(torch.cuda.current_stream(device).cuda_stream)


def rotary_axes(x, positions, sections: Sequence[int], *, base: float = 10000.0, ladder: str = "axis",
                frequencies: Optional[Sequence[float]] = None, pairs: str = "split", inverse: bool = False,
                out=None, stream=None):
    """Turn every pair of x's head dimension by position * frequency of the pair's axis (nerf_rotary_axes).

    x: [tokens, heads, dim] or [batch, tokens, heads, dim] of float32, bfloat16 or float16 with a
    contiguous last dimension (any other strides: heads before tokens is a transposed view), or a pair
    of such tensors (queries, keys) with the same batch, tokens, dim and type.  positions: [tokens, axes]
    (shared by the batch) or [batch, tokens, axes], float32, int32 or int64.  sections: pairs per axis,
    first the first axis's; values behind 2 * sum(sections) pass through.  The pair's frequency is
    base^(-j / sections[a]) for pair j of axis a (ladder "axis"), base^(-i / sum(sections)) for pair i of
    all ("shared"), or frequencies[i].  pairs: "split" (x[i], x[i + sum(sections)]) or "interleaved"
    (x[2i], x[2i + 1]).  inverse=True turns back, which is the gradient of the forward turn.
    Returns new tensors with x's strides, or out (x itself, or memory that does not overlap it)."""
    import torch

    single = isinstance(x, torch.Tensor)
    xs = (x,) if single else tuple(x)
    if not 1 <= len(xs) <= 2:
        raise ValueError(f"one or two tensors, got {len(xs)}")
    _check_plain(torch, positions=positions, **{f"x[{i}]": t for i, t in enumerate(xs)})
    outs = None
    if out is not None:
        outs = (out,) if single else tuple(out)
        if len(outs) != len(xs):
            raise ValueError(f"{len(xs)} outputs needed, got {len(outs)}")
        _check_plain(torch, **{f"out[{i}]": t for i, t in enumerate(outs)})
    first = xs[0]
    codes = _dtypes()
    if first.dtype not in codes:
        raise ValueError(f"x must be float32, bfloat16 or float16, got {first.dtype}")
    sections = [int(s) for s in sections]
    total = sum(sections)
    if not 1 <= len(sections) <= rt.NERF_ROTARY_MAX_AXES or min(sections) < 0:
        raise ValueError(f"sections {sections}: 1 to {rt.NERF_ROTARY_MAX_AXES} counts of pairs")
    if pairs not in PAIRS:
        raise ValueError(f"pairs {pairs!r}: one of {PAIRS}")
    if ladder not in LADDERS:
        raise ValueError(f"ladder {ladder!r}: one of {LADDERS}")
    if first.dim() not in (3, 4):
        raise ValueError(f"x must be [tokens, heads, dim] or [batch, tokens, heads, dim], got {tuple(first.shape)}")
    batched = first.dim() == 4
    batch = first.shape[0] if batched else 1
    tokens, dim = int(first.shape[-3]), int(first.shape[-1])
    if 2 * total > dim or total > rt.NERF_ROTARY_MAX_PAIRS:
        raise ValueError(f"sections {sections} hold {total} pairs: at most {min(dim // 2, rt.NERF_ROTARY_MAX_PAIRS)}")
    for i, t in enumerate(xs):
        if t.dim() != first.dim() or t.dtype != first.dtype or t.shape[:-2] != first.shape[:-2] or t.shape[-1] != dim:
            raise ValueError(f"x[{i}] {tuple(t.shape)} {t.dtype} does not go with x[0] {tuple(first.shape)} {first.dtype}")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"x[{i}]'s last dimension must be contiguous")
    shape = tuple(positions.shape)
    if shape not in ((tokens, len(sections)), (batch, tokens, len(sections))):
        raise ValueError(f"positions must be [{tokens}, {len(sections)}] or [{batch}, {tokens}, {len(sections)}], got {shape}")
    kinds = {torch.float32: rt.NERF_F32, torch.int32: rt.NERF_INT32, torch.int64: rt.NERF_INT64}
    if positions.dtype not in kinds:
        raise ValueError(f"positions must be float32, int32 or int64, got {positions.dtype}")
    if outs is not None:
        for i, (t, o) in enumerate(zip(xs, outs)):
            if o.shape != t.shape or o.dtype != t.dtype or (dim > 1 and o.stride(-1) != 1):
                raise ValueError(f"out[{i}] must have x[{i}]'s shape and type and a contiguous last dimension")
            if any(s == 0 and n > 1 for s, n in zip(o.stride(), o.shape)):
                raise ValueError(f"out[{i}] repeats its memory")
            if o.data_ptr() == t.data_ptr() and o.numel() and o.stride() != t.stride():
                raise ValueError(f"out[{i}] overlaps x[{i}] in another order")
        if len(outs) == 2 and outs[0].data_ptr() == outs[1].data_ptr() and outs[0].numel() and outs[1].numel():
            raise ValueError("the two outputs share their memory")
    d = rt.RotaryDesc()
    d.dtype, d.head_dim, d.n_axes = codes[first.dtype], dim, len(sections)
    d.sections[:len(sections)] = sections
    d.shared_ladder, d.interleaved, d.inverse = ladder == "shared", pairs == "interleaved", bool(inverse)
    d.base = float(base)
    if frequencies is not None:
        table = [float(f) for f in frequencies]
        if len(table) != total:
            raise ValueError(f"{total} frequencies needed, got {len(table)}")
        d.frequencies = (ctypes.c_double * total)(*table)
    stride = positions.stride()
    d.position_stride[:] = stride if len(shape) == 3 else (0, *stride)
    d.position_dtype, d.n_batch, d.n_tokens, d.n_tensors = kinds[positions.dtype], batch, tokens, len(xs)
    named = {f"x[{i}]": t for i, t in enumerate(xs)}
    named.update({f"out[{i}]": t for i, t in enumerate(outs or ())})
    with _On(torch, first.device, stream, positions=positions, **named) as on:
        if outs is None:
            outs = tuple(torch.empty_like(t) for t in xs)
        d.positions = positions.data_ptr()
        for k, (t, o) in enumerate(zip(xs, outs)):
            e = d.tensor[k]
            e.x, e.out, e.heads = t.data_ptr(), o.data_ptr(), t.shape[-2]
            e.x_stride[:] = t.stride()[:3] if batched else (0, *t.stride()[:2])
            e.out_stride[:] = o.stride()[:3] if batched else (0, *o.stride()[:2])
        rt._check(rt.load_library().nerf_rotary_axes(ctypes.byref(d), on.stream))
    return outs[0] if single else outs


def _rows(t, name: str, width: int):
    """t [..., width] as [rows, width] without a copy, and its row stride."""
    if t.dim() < 1 or t.shape[-1] != width:
        raise ValueError(f"{name} must be [..., {width}], got {tuple(t.shape)}")
    if width > 1 and t.stride(-1) != 1 and t.numel():
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if t.dim() != 2:
        try:
            t = t.view(-1, width) if t.numel() else t.reshape(0, width)
        except RuntimeError:
            raise ValueError(f"{name} {tuple(t.shape)} with strides {t.stride()} is not rows of one stride") from None
    stride = t.stride(0) if t.shape[0] > 1 else max(t.stride(0), width)
    if stride < width:
        raise ValueError(f"{name}'s rows overlap (stride {stride}, width {width})")
    return t, stride


def _block(torch, x, w_gate, w_up, w_down, activation):
    _check_plain(torch, x=x, w_gate=w_gate, w_up=w_up, w_down=w_down)
    codes = _dtypes()
    if x.dtype not in codes:
        raise ValueError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: one of {tuple(ACTIVATIONS)}")
    for name, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if w.dim() != 2 or w.dtype != x.dtype or 0 in w.shape:
            raise ValueError(f"{name} must be a matrix of x's type {x.dtype}, got {tuple(w.shape)} {w.dtype}")
    hidden, width = w_gate.shape
    if w_up.shape != w_gate.shape or w_down.shape[1] != hidden:
        raise ValueError(f"w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and w_down {tuple(w_down.shape)} must be "
                         "[hidden, width], [hidden, width] and [out, hidden]")
    d = rt.BlockDesc()
    x2, d.ld_x = _rows(x, "x", width)
    for name, w, n in (("gate", w_gate, width), ("up", w_up, width), ("down", w_down, hidden)):
        setattr(d, f"ld_{name}", _rows(w, f"w_{name}", n)[1])
    d.dtype, d.activation = codes[x.dtype], ACTIVATIONS[activation]
    d.rows, d.width, d.hidden, d.out = x2.shape[0], width, hidden, w_down.shape[0]
    d.x, d.w_gate, d.w_up, d.w_down = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr()
    return d


def _workspace(torch, d, backward: int, device):
    n = rt.load_library().nerf_gated_block_workspace(ctypes.byref(d), backward)
    return torch.empty(max(n, 1), dtype=torch.uint8, device=device), n


def gated_block(x, w_gate, w_up, w_down, *, activation: str = "silu", out=None, stream=None):
    """y = (act(x w_gate^T) * (x w_up^T)) w_down^T  (nerf_gated_block_forward).

    x: [..., width]; w_gate, w_up: [hidden, width]; w_down: [out, hidden]; one type, float32, bfloat16 or
    float16, last dimensions contiguous, any row strides.  activation: "silu", "gelu" (x Phi(x)) or
    "relu".  Sums are held in 32 bits; the hidden row is rounded once for the 16-bit types.  Returns
    [..., out], or writes out (rows of one stride that overlap no input)."""
    import torch

    d = _block(torch, x, w_gate, w_up, w_down, activation)
    shape = (*x.shape[:-1], d.out)
    if out is not None:
        _check_plain(torch, out=out)
        if tuple(out.shape) != shape or out.dtype != x.dtype:
            raise ValueError(f"out must be {shape} {x.dtype}, got {tuple(out.shape)} {out.dtype}")
    named = dict(w_gate=w_gate, w_up=w_up, w_down=w_down, **({} if out is None else {"out": out}))
    with _On(torch, x.device, stream, **named) as on:
        y = torch.empty(shape, dtype=x.dtype, device=x.device) if out is None else out
        _, ld = _rows(y, "out", d.out)
        _refuse_overlap(dict(out=y), dict(x=x, w_gate=w_gate, w_up=w_up, w_down=w_down))
        ws, n = _workspace(torch, d, 0, x.device)
        rt._check(rt.load_library().nerf_gated_block_forward(ctypes.byref(d), y.data_ptr(), ld, ws.data_ptr(), n, on.stream))
    return y


def gated_block_backward(dy, x, w_gate, w_up, w_down, *, activation: str = "silu",
                         needs: Sequence[bool] = (True, True, True, True), out=(None, None, None, None), stream=None):
    """The gradients (dx, dw_gate, dw_up, dw_down) of gated_block for dy = dL/dy (nerf_gated_block_backward).

    The pre-activations are recomputed from x: the forward call keeps nothing.  needs: which of the four
    to compute (the others are None); out: where to write them (new tensors for None); the weights'
    gradients are contiguous."""
    import torch

    d = _block(torch, x, w_gate, w_up, w_down, activation)
    _check_plain(torch, dy=dy)
    if dy.shape[:-1] != x.shape[:-1] or dy.dtype != x.dtype:
        raise ValueError(f"dy {tuple(dy.shape)} {dy.dtype} does not go with x {tuple(x.shape)} {x.dtype}")
    _, ld_dy = _rows(dy, "dy", d.out)
    if len(needs) != 4 or len(out) != 4:
        raise ValueError("needs and out have four entries: dx, dw_gate, dw_up, dw_down")
    names, likes = ("dx", "dw_gate", "dw_up", "dw_down"), (x, w_gate, w_up, w_down)
    given = {k: o for k, o, n in zip(names, out, needs) if n and o is not None}
    _check_plain(torch, **given)
    for k, o in given.items():
        like = likes[names.index(k)]
        if o.shape != like.shape or o.dtype != like.dtype or (k != "dx" and not o.is_contiguous()):
            raise ValueError(f"{k} must be {tuple(like.shape)} {like.dtype}" + (", contiguous" if k != "dx" else ""))
    inputs = dict(dy=dy, x=x, w_gate=w_gate, w_up=w_up, w_down=w_down)
    with _On(torch, x.device, stream, **{k: v for k, v in inputs.items() if k != "x"}, **given) as on:
        got = [None if not n else given.get(k) if k in given else
               torch.empty(like.shape, dtype=like.dtype, device=like.device) for k, like, n in zip(names, likes, needs)]
        _refuse_overlap({k: g for k, g in zip(names, got) if g is not None}, inputs)
        ld_dx = _rows(got[0], "dx", d.width)[1] if got[0] is not None else d.width
        ws, n = _workspace(torch, d, 1, x.device)
        ptr = [None if g is None else g.data_ptr() for g in got]
        rt._check(rt.load_library().nerf_gated_block_backward(ctypes.byref(d), dy.data_ptr(), ld_dy, ptr[0], ld_dx, ptr[1],
                                                              ptr[2], ptr[3], ws.data_ptr(), n, on.stream))
    return tuple(got)


def _span(t):
    """The byte range [first, last) a tensor's values lie in."""
    if not t.numel():
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _refuse_overlap(outputs, inputs) -> None:
    spans = {k: _span(t) for k, t in inputs.items()}
    for name, t in outputs.items():
        a, b = _span(t)
        for other, (c, e) in spans.items():
            if a < e and c < b:
                raise ValueError(f"{name} overlaps {other} in memory")
        spans[name] = (a, b)
