"""Operators of sequence models: the gated linear recurrence (a conv1d whose filter changes from sample to
sample), the gated linear layer, and products of few rows with 4-bit weights.

GPU tensors run the native HIP kernels; CPU tensors run the definitions in float64.  Arguments are checked on both.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._util import launch, plain_tensors, records

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 5}


def _opt(t):
    return None if t is None else t.data_ptr()


def _rows_last(t: torch.Tensor) -> torch.Tensor:
    """t with neighbouring elements in its last dimension (a copy only where they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _same_device(name, first, **others):
    for n, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name}: {n} is on {t.device}, x on {first.device}")


def _new(x: torch.Tensor, *shape) -> torch.Tensor:
    return x.new_empty(shape)


# ------------------------------------------------------- gated recurrence
def _check_recurrence(name, x, gate, state, lengths):
    if x.dtype not in DTYPES:
        raise TypeError(f"{name}: x is {x.dtype}; float32, float16 or bfloat16 expected")
    if gate.dtype != x.dtype:
        raise TypeError(f"{name}: gate is {gate.dtype}, x {x.dtype}")
    if x.dim() != 3 or gate.shape != x.shape:
        raise ValueError(f"{name}: x and gate are [batch, time, channels]; got {tuple(x.shape)} and "
                         f"{tuple(gate.shape)}")
    if state is not None:
        if state.dtype != torch.float32:
            raise TypeError(f"{name}: the state is float32; got {state.dtype}")
        if tuple(state.shape) != (x.shape[0], x.shape[2]):
            raise ValueError(f"{name}: state {tuple(state.shape)}, [batch, channels] = "
                             f"{(x.shape[0], x.shape[2])} expected")
    if lengths is not None:
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name}: lengths are int32 or int64; got {lengths.dtype}")
        if tuple(lengths.shape) != (x.shape[0],):
            raise ValueError(f"{name}: lengths {tuple(lengths.shape)}, one per sequence "
                             f"({x.shape[0]}) expected")
    _same_device(name, x, gate=gate, state=state, lengths=lengths)


def _tiles(t):
    """vs_gated_recurrence_tiles(t), in arithmetic that a symbolic length passes through."""
    return (t + 127) // 128


def _recurrence_workspace(x):
    size = int(_lib.lib().vs_gated_recurrence_workspace(*x.shape))
    return torch.empty(size, dtype=torch.uint8, device=x.device) if size else None


def _valid_steps(x, lengths):
    n = torch.full((x.shape[0],), x.shape[1], device=x.device) if lengths is None else lengths.clamp(0, x.shape[1])
    return torch.arange(x.shape[1], device=x.device)[:, None] < n[None, :]      # [time, batch]


def _recurrence_cpu(x, gate, state, lengths, save):
    b, t, d = x.shape
    on = _valid_steps(x, lengths)
    h = x.new_zeros(b, d, dtype=torch.float64) if state is None else state.double()
    xd, i, keep = x.double(), torch.sigmoid(-gate.double()), torch.sigmoid(gate.double())
    y = x.new_zeros(b, t, d, dtype=torch.float64)
    for s in range(t):
        h = torch.where(on[s][:, None], keep[:, s] * h + i[:, s] * xd[:, s], h)
        y[:, s] = torch.where(on[s][:, None], h, 0.0)
    # the CPU backward starts from the initial state: one tile
    starts = (x.new_zeros(b, d, dtype=torch.float32) if state is None else state)[:, None].clone() if save else None
    return y.to(x.dtype), h.float(), starts


def _recurrence_impl(x, gate, state, lengths, save):
    _check_recurrence("veles::gated_recurrence", x, gate, state, lengths)
    if not x.is_cuda:
        return _recurrence_cpu(x, gate, state, lengths, save)
    b, t, d = x.shape
    x, gate = _rows_last(x), _rows_last(gate)
    state = None if state is None else state.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    y = torch.empty((b, t, d), dtype=x.dtype, device=x.device)
    final = torch.empty((b, d), dtype=torch.float32, device=x.device)
    starts = torch.empty((b, _tiles(t), d), dtype=torch.float32, device=x.device) if save else None
    ws = _recurrence_workspace(x)
    launch(x, "vs_gated_recurrence", DTYPES[x.dtype], x.data_ptr(), x.stride(0), x.stride(1), gate.data_ptr(),
           gate.stride(0), gate.stride(1), _opt(state), _opt(lengths),
           int(lengths is not None and lengths.dtype == torch.int64), b, t, d, y.data_ptr(), final.data_ptr(),
           _opt(starts), _opt(ws), 0 if ws is None else ws.numel())
    return y, final, starts


def _recurrence_backward_cpu(x, gate, lengths, starts, dy, dfinal):
    b, t, d = x.shape
    on = _valid_steps(x, lengths)
    xd, i, keep = x.double(), torch.sigmoid(-gate.double()), torch.sigmoid(gate.double())
    h = starts[:, 0].double()
    before = x.new_zeros(b, t, d, dtype=torch.float64)
    for s in range(t):
        before[:, s] = h
        h = torch.where(on[s][:, None], keep[:, s] * h + i[:, s] * xd[:, s], h)
    m = x.new_zeros(b, d, dtype=torch.float64) if dfinal is None else dfinal.double()
    dx, dg = (x.new_zeros(b, t, d, dtype=torch.float64) for _ in range(2))
    for s in range(t - 1, -1, -1):
        k = on[s][:, None]
        lam = m if dy is None else m + dy[:, s].double()
        dx[:, s] = torch.where(k, i[:, s] * lam, 0.0)
        dg[:, s] = torch.where(k, i[:, s] * keep[:, s] * lam * (before[:, s] - xd[:, s]), 0.0)
        m = torch.where(k, keep[:, s] * lam, m)
    return dx.to(x.dtype), dg.to(x.dtype), m.float()


def _recurrence_backward_impl(x, gate, lengths, starts, dy, dfinal):
    name = "veles::gated_recurrence_backward"
    _check_recurrence(name, x, gate, dfinal, lengths)
    if dy is not None and (dy.shape != x.shape or dy.dtype != x.dtype):
        raise ValueError(f"{name}: dy is {dy.dtype} {tuple(dy.shape)}, {x.dtype} {tuple(x.shape)} expected")
    if starts.dtype != torch.float32:
        raise TypeError(f"{name}: the saved states are float32; got {starts.dtype}")
    _same_device(name, x, starts=starts, dy=dy)
    b, t, d = x.shape
    want = (b, _tiles(t) if x.is_cuda else 1, d)
    if tuple(starts.shape) != want:
        raise ValueError(f"{name}: saved states {tuple(starts.shape)}, {want} expected")
    if not x.is_cuda:
        return _recurrence_backward_cpu(x, gate, lengths, starts, dy, dfinal)
    x, gate = _rows_last(x), _rows_last(gate)
    dy = None if dy is None else _rows_last(dy)
    dfinal = None if dfinal is None else dfinal.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    starts = starts.contiguous()
    dx = torch.empty((b, t, d), dtype=x.dtype, device=x.device)
    dg = torch.empty_like(dx)
    dstate = torch.empty((b, d), dtype=torch.float32, device=x.device)
    ws = _recurrence_workspace(x)
    launch(x, "vs_gated_recurrence_backward", DTYPES[x.dtype], x.data_ptr(), x.stride(0), x.stride(1),
           gate.data_ptr(), gate.stride(0), gate.stride(1), _opt(lengths),
           int(lengths is not None and lengths.dtype == torch.int64), starts.data_ptr(), _opt(dy),
           0 if dy is None else dy.stride(0), 0 if dy is None else dy.stride(1), _opt(dfinal), b, t, d,
           dx.data_ptr(), dg.data_ptr(), dstate.data_ptr(), _opt(ws), 0 if ws is None else ws.numel())
    return dx, dg, dstate


def _recurrence_fake(x, gate, state, lengths, save):
    _check_recurrence("veles::gated_recurrence", x, gate, state, lengths)
    b, t, d = x.shape
    starts = (b, _tiles(t) if x.is_cuda else 1, d) if save else (0,)
    return (x.new_empty((b, t, d)), x.new_empty((b, d), dtype=torch.float32),
            x.new_empty(starts, dtype=torch.float32))


def _recurrence_setup(ctx, inputs, output):
    x, gate, state, lengths, save = inputs
    if not save:
        raise RuntimeError("veles::gated_recurrence: gradients need the saved states (save=True)")
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(output[2])
    ctx.save_for_backward(x, gate, lengths, output[2])


def _recurrence_grad(ctx, dy, dfinal, _):
    return *_recurrence_grads(ctx, torch.ops.veles.gated_recurrence_backward, dy, dfinal), None, None


def _recurrence_grads(ctx, backward, dy, dfinal):
    if dy is None and dfinal is None:
        return None, None, None
    x, gate, lengths, starts = ctx.saved_tensors
    dx, dg, dstate = backward(x, gate, lengths, starts, dy, dfinal)
    need = ctx.needs_input_grad
    return dx if need[0] else None, dg if need[1] else None, dstate if need[2] else None


class _Recurrence(torch.autograd.Function):
    """The op's autograd without the dispatcher."""

    @staticmethod
    def forward(ctx, x, gate, state, lengths):
        y, final, starts = _recurrence_impl(x, gate, state, lengths, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, gate, lengths, starts)
        return y, final

    @staticmethod
    def backward(ctx, dy, dfinal):
        # a graph of the gradients asks for second derivatives, which the op refuses by name
        op = torch.ops.veles.gated_recurrence_backward if torch.is_grad_enabled() else _recurrence_backward_impl
        return *_recurrence_grads(ctx, op, dy, dfinal), None


def _with_empty(impl):
    """impl for the dispatcher: what is not saved (None, last) becomes an empty float32 tensor."""
    def op(x, *args):
        *out, saved = impl(x, *args)
        return (*out, x.new_empty(0, dtype=torch.float32) if saved is None else saved)
    return op


def _no_second_derivative(name):
    def setup(ctx, inputs, output):
        pass

    def grad(ctx, *_):
        raise NotImplementedError(f"{name} has no derivative of its own (second derivatives)")
    torch.library.register_autograd(name, grad, setup_context=setup)


torch.library.define("veles::gated_recurrence",
                     "(Tensor x, Tensor gate, Tensor? state, Tensor? lengths, bool save) -> (Tensor, Tensor, Tensor)")
torch.library.impl("veles::gated_recurrence", "default", _with_empty(_recurrence_impl))
torch.library.register_fake("veles::gated_recurrence", _recurrence_fake)
torch.library.register_autograd("veles::gated_recurrence", _recurrence_grad, setup_context=_recurrence_setup)
torch.library.define("veles::gated_recurrence_backward",
                     "(Tensor x, Tensor gate, Tensor? lengths, Tensor starts, Tensor? dy, Tensor? dfinal) -> "
                     "(Tensor, Tensor, Tensor)")
torch.library.impl("veles::gated_recurrence_backward", "default", _recurrence_backward_impl)
torch.library.register_fake(
    "veles::gated_recurrence_backward",
    lambda x, gate, lengths, starts, dy, dfinal: (
        x.new_empty(x.shape), x.new_empty(x.shape),
        x.new_empty((x.shape[0], x.shape[2]), dtype=torch.float32)))
_no_second_derivative("veles::gated_recurrence_backward")


def gated_recurrence(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None):
    """Gated linear recurrence along time, (y, final_state):

        i_t = sigmoid(-gate_t),  h_t = (1 - i_t) h_{t-1} + i_t x_t,  y_t = h_t

    x, gate: [batch, time, channels], float32, float16 or bfloat16, any batch and time strides.
    state: h_0, float32 [batch, channels] (zeros if None); final_state is the float32 state after
    the last step, so a sequence can be continued by another call or by gated_recurrence_step.
    lengths: int32 / int64 [batch] on x's device: steps from lengths[b] on are padding (not read,
    y = 0, the state passes through; values outside 0..time are clamped).
    The state is held in float32, and i and 1 - i have all of float32's digits for every gate.  Differentiable
    in x, gate and state; in the padding the gradients are 0 and dy is not read.  From an infinite state or
    value on, a channel is infinite or NaN to its end."""
    save = records(x, gate, state)
    if plain_tensors(x, gate, state, lengths):
        if save:
            return _Recurrence.apply(x, gate, state, lengths)
        return _recurrence_impl(x, gate, state, lengths, False)[:2]
    y, final, _ = torch.ops.veles.gated_recurrence(x, gate, state, lengths, save)
    return y, final


def _check_step(x, gate, state):
    name = "veles::gated_recurrence_step"
    for t in (x, gate):
        if t.dim() != 2:
            raise ValueError(f"{name}: x and gate are [batch, channels]; got {tuple(t.shape)}")
    _check_recurrence(name, x[:, None], gate[:, None], state, None)
    if not state.is_contiguous():
        raise ValueError(f"{name}: the state is updated in place and has to be contiguous")


def _overlaps(p, ld, t, state):
    """Whether rows t, at address p, lie in the memory of the state of their shape in another place than the state's
    own values, so that a step would read what it writes elsewhere."""
    b, d = t.shape
    return p < state + 4 * b * d and p + ((b - 1) * ld + d) * t.itemsize > state \
        and not (p == state and ld == d and t.itemsize == 4)


def _step_impl(x, gate, state):
    # the usual case in one expression; _check_step names what is wrong otherwise
    if not (x.dim() == 2 and x.shape == gate.shape == state.shape and x.dtype is gate.dtype
            and x.dtype in DTYPES and state.dtype is torch.float32 and state.is_contiguous()
            and x.device == gate.device == state.device):
        _check_step(x, gate, state)
    if not x.is_cuda:
        g = gate.double()
        state.copy_(torch.sigmoid(g) * state + torch.sigmoid(-g) * x)
        return state.to(x.dtype, copy=True)
    b, d = x.shape
    if x.is_contiguous() and gate.is_contiguous():
        y, ldx, ldg = torch.empty_like(x), d, d
    else:
        x, gate = _rows_last(x), _rows_last(gate)
        y, ldx, ldg = _new(x, b, d), x.stride(0), gate.stride(0)
    px, pg, ps = x.data_ptr(), gate.data_ptr(), state.data_ptr()
    size = 4 * b * d    # rows one behind the other and this far from the state cannot reach it
    if (-size < px - ps < size or -size < pg - ps < size or ldx != d or ldg != d) \
            and (_overlaps(px, ldx, x, ps) or _overlaps(pg, ldg, gate, ps)):
        x, gate = x.clone(), gate.clone()   # (kept until the launch)
        px, ldx, pg, ldg = x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0)
    launch(x, "vs_gated_recurrence_step", DTYPES[x.dtype], px, ldx, pg, ldg, ps, b, d, y.data_ptr())
    return y


torch.library.define("veles::gated_recurrence_step", "(Tensor x, Tensor gate, Tensor(a!) state) -> Tensor")
torch.library.impl("veles::gated_recurrence_step", "default", _step_impl)
torch.library.register_fake("veles::gated_recurrence_step", lambda x, gate, state: x.new_empty(x.shape))


def gated_recurrence_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
    """One step of gated_recurrence for a batch of sequences: x, gate [batch, channels]; state
    (float32 [batch, channels], contiguous) is updated in place and returned as y in x's type.
    For generation: it records no gradient."""
    if records(x, gate, state):
        raise RuntimeError("gated_recurrence_step records no gradient: call it under torch.no_grad(), or use "
                           "gated_recurrence")
    if plain_tensors(x, gate, state):
        y = _step_impl(x, gate, state)
        if not state.is_inference():
            torch.autograd.graph.increment_version(state)   # as the dispatcher does for an op that writes
        return y
    return torch.ops.veles.gated_recurrence_step(x, gate, state)


# -------------------------------------------------------- 4-bit products
def _check_group(name, group_size):
    if group_size not in (32, 64) and (group_size <= 0 or group_size % 128):
        raise ValueError(f"{name}: group size {group_size}; 32, 64 or a multiple of 128 expected")


_HALF = (torch.float16, torch.bfloat16)


def _check_matvec(name, x, qweight, scales, zeros, group_size):
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name}: x is {x.dtype}; float16 or bfloat16 expected")
    if x.dim() < 1 or qweight.dim() != 2 or qweight.dtype != torch.uint8:
        raise ValueError(f"{name}: x [..., k] and uint8 qweight [n, (k + 1) // 2] expected")
    _check_group(name, group_size)
    n, k = qweight.shape[0], x.shape[-1]
    if qweight.shape[1] != (k + 1) // 2:
        raise ValueError(f"{name}: qweight {tuple(qweight.shape)} does not fit x with {k} columns")
    groups = (n, -(-k // group_size))
    if scales.dtype != x.dtype:
        raise TypeError(f"{name}: scales are {scales.dtype}, x {x.dtype}")
    if scales.shape != groups:
        raise ValueError(f"{name}: scales {tuple(scales.shape)}, {groups} expected")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != groups):
        raise ValueError(f"{name}: zeros {zeros.dtype} {tuple(zeros.shape)}, uint8 {groups} expected")
    if (qweight.shape[1] > 1 and qweight.stride(1) != 1) or (n > 1 and qweight.stride(0) < qweight.shape[1]):
        raise ValueError(f"{name}: the bytes of a row of qweight have to be neighbours and rows apart")
    _same_device(name, x, qweight=qweight, scales=scales, zeros=zeros)


def _matvec_impl(x, qweight, scales, zeros, group_size):
    name = "veles::matvec_int4"
    # the usual case in one expression; _check_matvec names what is wrong otherwise
    dev, dtype = x.get_device(), x.dtype
    if (dev >= 0 and x.dim() == 2 and qweight.dim() == 2 and dtype in _HALF and scales.dtype is dtype
            and qweight.dtype is torch.uint8 and (group_size in (32, 64) or (group_size > 0 and group_size % 128 == 0))
            and x.is_contiguous() and qweight.is_contiguous() and scales.is_contiguous()
            and dev == qweight.get_device() == scales.get_device()
            and (zeros is None or (zeros.dtype is torch.uint8 and zeros.is_contiguous()
                                   and zeros.shape == scales.shape and dev == zeros.get_device()))):
        (m, k), (n, half) = x.shape, qweight.shape
        if half == (k + 1) // 2 and scales.shape == (n, -(-k // group_size)):
            y = x.new_empty((m, n))
            launch(x, "vs_matvec_int4", DTYPES[dtype], x.data_ptr(), k, qweight.data_ptr(), half, scales.data_ptr(),
                   _opt(zeros), group_size, m, n, k, y.data_ptr())
            return y
    _check_matvec(name, x, qweight, scales, zeros, group_size)
    n, k = qweight.shape[0], x.shape[-1]
    if not x.is_cuda:
        q = torch.stack([qweight & 15, qweight >> 4], -1).flatten(1)[:, :k].double()
        at = torch.arange(k, device=x.device) // group_size
        z = 8.0 if zeros is None else zeros.double()[:, at]
        return (x.double() @ ((q - z) * scales.double()[:, at]).t()).to(x.dtype)
    rows = _near_rows(_as_rows(x), True)
    y = _new(x, *x.shape[:-1], n)
    scales = scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    launch(x, "vs_matvec_int4", DTYPES[x.dtype], rows.data_ptr(), rows.stride(0), qweight.data_ptr(),
           qweight.stride(0), scales.data_ptr(), _opt(zeros), group_size, rows.shape[0], n, k, y.data_ptr())
    return y


def _matvec_fake(x, qweight, scales, zeros, group_size):
    _check_matvec("veles::matvec_int4", x, qweight, scales, zeros, group_size)
    return x.new_empty((*x.shape[:-1], qweight.shape[0]))


torch.library.define("veles::matvec_int4",
                     "(Tensor x, Tensor qweight, Tensor scales, Tensor? zeros, int group_size) -> Tensor")
torch.library.impl("veles::matvec_int4", "default", _matvec_impl)
torch.library.register_fake("veles::matvec_int4", _matvec_fake)


def matvec_int4(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor,
                zeros: torch.Tensor | None = None, group_size: int = 128) -> torch.Tensor:
    """x @ W.T for few rows x [..., k] (float16 or bfloat16) and a weight kept in 4 bits:

        W[n, j] = (q[n, j] - zeros[n, j // group_size]) * scales[n, j // group_size]

    qweight: uint8 [n, (k + 1) // 2], two numbers 0..15 to a byte, the even column in the low half.
    scales: x's type, [n, ceil(k / group_size)]; zeros: uint8 of that shape (8 everywhere if None).
    group_size: 32, 64 or a multiple of 128; the last group may end early.  Weights are exact and sums
    are float32; the result is rounded once, to x's type.  On a GPU the zero points are taken off the sums, so
    float32's rounding is relative to sum |x| (32 + q + zeros) scales, also where q is close to zeros, and x has to be
    finite, with sums of 2 |x| (or (1 + zeros / 16) |x|, where that is more) over a group below 3.4e38.
    For generation: it records no gradient; more than 16 rows read the weights once for every 16.
    quantize_int4 makes the operands."""
    if records(x, scales):
        raise RuntimeError("matvec_int4 records no gradient: call it under torch.no_grad()")
    if plain_tensors(x, qweight, scales, zeros):
        return _matvec_impl(x, qweight, scales, zeros, group_size)
    return torch.ops.veles.matvec_int4(x, qweight, scales, zeros, group_size)


def quantize_int4(weight: torch.Tensor, group_size: int = 128, symmetric: bool = False,
                  dtype: torch.dtype | None = None):
    """(qweight, scales, zeros) of a weight [n, k] for matvec_int4, to be made once and kept.  Every
    group's range, zero included, is cut into 15 steps (symmetric: +-7 steps around 8, zeros None).
    dtype: of the scales, the type that x will have (weight's, or bfloat16 for a float32 weight)."""
    _check_group("quantize_int4", group_size)
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"quantize_int4: a floating weight [n, k] expected; got {weight.dtype} {tuple(weight.shape)}")
    dtype = dtype or (weight.dtype if weight.dtype in (torch.float16, torch.bfloat16) else torch.bfloat16)
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"quantize_int4: scales of {dtype}; float16 or bfloat16 expected")
    w = weight.detach().float()
    if not torch.isfinite(w).all():
        raise ValueError("quantize_int4: the weight has values that are not finite")
    n, k = w.shape
    groups = -(-k // group_size)
    w = torch.nn.functional.pad(w, (0, groups * group_size - k)).view(n, groups, group_size)
    if symmetric:
        step = w.abs().amax(-1) / 7 if groups else w.new_zeros(n, 0)
    else:
        lo, hi = (w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)) if groups else (w.new_zeros(n, 0),) * 2
        step = (hi - lo) / 15
    scales = step.to(dtype)
    if not torch.isfinite(scales).all():
        raise ValueError(f"quantize_int4: a group's step does not fit {dtype}")
    step = scales.float()
    step = torch.where(step > 0, step, 1.0)
    zeros = torch.full_like(step, 8.0) if symmetric else torch.round(-lo / step).clamp(0, 15)
    q = torch.clamp(torch.round(w / step[..., None]) + zeros[..., None], 0, 15).to(torch.uint8)
    q = torch.nn.functional.pad(q.view(n, -1)[:, :k], (0, k % 2))
    return q[:, 0::2] | (q[:, 1::2] << 4), scales, None if symmetric else zeros.to(torch.uint8)


# ---------------------------------------------------- gated linear layer
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


def _check_gated(name, x, w_gate, w_up, activation):
    if activation not in ACTIVATIONS:
        raise ValueError(f"{name}: activation {activation!r}; one of {sorted(ACTIVATIONS)} expected")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name}: x is {x.dtype}; float16 or bfloat16 expected")
    if w_gate.dtype != x.dtype or w_up.dtype != x.dtype:
        raise TypeError(f"{name}: weights are {w_gate.dtype} and {w_up.dtype}, x {x.dtype}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_gate.shape[1] != x.shape[-1]:
        raise ValueError(f"{name}: x [..., k] and two weights [features, k] expected; got {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)}, {tuple(w_up.shape)}")
    _same_device(name, x, w_gate=w_gate, w_up=w_up)


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., k] as [rows, k] with neighbouring k (a copy only where the layout asks for one)."""
    if x.dim() != 2:
        rows = 1
        for n in x.shape[:-1]:
            rows *= n
        x = x.reshape(rows, x.shape[-1])
    return _rows_last(x)


_LD_MAX = 1 << 21   # the tile kernel keeps 32-bit offsets over 256 rows


def _near_rows(t: torch.Tensor, shared: bool) -> torch.Tensor:
    """[rows, k] with a row stride that the kernels take: at least k (or 0 if `shared`), below _LD_MAX."""
    t = _rows_last(t)
    ld = t.stride(0)
    if ld < _LD_MAX and (ld >= t.shape[1] or t.shape[0] <= 1 or (shared and ld == 0)):
        return t
    return t.contiguous() if t.shape[0] > 1 else t.reshape(-1).view(t.shape)


def _act_cpu(kind, g):
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return 0.5 * g * torch.special.erfc(g * -0.5 ** 0.5)
    return torch.relu(g) if kind == "relu" else torch.sigmoid(g)


def _slope_cpu(kind, g):
    s = torch.sigmoid(g)
    if kind == "silu":
        return s * (1.0 + g * (1.0 - s))
    if kind == "gelu":
        return 0.5 * torch.special.erfc(g * -0.5 ** 0.5) + g * torch.exp(-0.5 * g * g) * (0.5 / torch.pi) ** 0.5
    return (g > 0).to(g.dtype) if kind == "relu" else s * torch.sigmoid(-g)


def _gated_impl(x, w_gate, w_up, activation, save, split=False):
    name = "veles::gated_linear"
    # few rows, as a generating model has them, in one expression; _check_gated names what is wrong otherwise
    dev, dtype = x.get_device(), x.dtype
    if (dev >= 0 and not save and x.dim() == 2 and w_gate.dim() == 2 and dtype in _HALF
            and w_gate.dtype is dtype and w_up.dtype is dtype and activation in ACTIVATIONS
            and x.is_contiguous() and w_gate.is_contiguous() and w_up.is_contiguous()
            and dev == w_gate.get_device() == w_up.get_device()):
        (m, k), (f, kw) = x.shape, w_gate.shape
        if m <= 16 and k == kw < _LD_MAX and w_up.shape == w_gate.shape:
            h = x.new_empty((m, f))
            launch(x, "vs_gated_linear", DTYPES[dtype], ACTIVATIONS[activation], x.data_ptr(), k, w_gate.data_ptr(), k,
                   w_up.data_ptr(), k, m, f, k, h.data_ptr(), None, None, 0)
            return h, None
    _check_gated(name, x, w_gate, w_up, activation)
    f, k = w_gate.shape
    rows = _near_rows(_as_rows(x), True)
    m = rows.shape[0]
    if save and split and (f > 1 << 19 or m >= (1 << 30) - 256):
        raise ValueError(f"{name}: split gradients of {m} rows and {f} features; 2^30 - 257 and 2^19 at most")
    if not x.is_cuda:
        g, u = rows.double() @ w_gate.double().t(), rows.double() @ w_up.double().t()
        h = (_act_cpu(activation, g) * u).to(x.dtype).view(*x.shape[:-1], f)
        return h, torch.stack([g, u], -1).float() if save else None
    w_gate, w_up = _near_rows(w_gate, False), _near_rows(w_up, False)
    h = _new(x, *x.shape[:-1], f)
    pre = torch.empty((m, f, 2), dtype=torch.float32, device=x.device) if save else None
    size, ws = 0, None
    if m > 16:      # fewer rows need none
        size = int(_lib.lib().vs_gated_linear_workspace(m, f, k, _aligned(rows, w_gate, w_up)))
        ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    launch(x, "vs_gated_linear", DTYPES[x.dtype], ACTIVATIONS[activation], rows.data_ptr(), rows.stride(0),
           w_gate.data_ptr(), w_gate.stride(0), w_up.data_ptr(), w_up.stride(0), m, f, k, h.data_ptr(),
           _opt(pre), _opt(ws), size)
    return h, pre


def _aligned(*tensors) -> bool:
    """Rows of whole 16-byte pieces: the kernel reads them where they are."""
    return all(t.shape[-1] % 8 == 0 and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0 for t in tensors)


def _gated_backward_impl(x, w_gate, w_up, pre, dh, activation, want_dx, want_dw_gate, want_dw_up=None, split=False):
    want_dw_up = want_dw_gate if want_dw_up is None else want_dw_up
    name = "veles::gated_linear_backward"
    _check_gated(name, x, w_gate, w_up, activation)
    f, k = w_gate.shape
    rows, dhr = _near_rows(_as_rows(x), True), _near_rows(_as_rows(dh), True)
    m = rows.shape[0]
    if dh.dtype != x.dtype or tuple(dh.shape) != (*x.shape[:-1], f):
        raise ValueError(f"{name}: dh is {dh.dtype} {tuple(dh.shape)}, {x.dtype} {(*x.shape[:-1], f)} expected")
    if pre.dtype != torch.float32 or tuple(pre.shape) != (m, f, 2):
        raise ValueError(f"{name}: pre-activations {pre.dtype} {tuple(pre.shape)}, float32 {(m, f, 2)} expected")
    _same_device(name, x, pre=pre, dh=dh)
    if not x.is_cuda:
        g, u, d = pre[..., 0].double(), pre[..., 1].double(), dhr.double()
        dg, du = d * u * _slope_cpu(activation, g), d * _act_cpu(activation, g)
        dx = (dg @ w_gate.double() + du @ w_up.double()).to(x.dtype).view(x.shape) if want_dx else x.new_empty(0)
        return dx, *((v.t() @ rows.double()).to(x.dtype) if want else x.new_empty(0)
                     for v, want in ((dg, want_dw_gate), (du, want_dw_up)))
    w_gate, w_up, pre = _near_rows(w_gate, False), _near_rows(w_up, False), pre.contiguous()
    dx = torch.empty(x.shape if want_dx else (0,), dtype=x.dtype, device=x.device)
    dwg, dwu = (torch.empty((f, k) if want else (0,), dtype=x.dtype, device=x.device)
                for want in (want_dw_gate, want_dw_up))
    aligned = (w_gate.stride(0) == w_up.stride(0) >= k <= rows.stride(0)) and _aligned(rows, w_gate, w_up)
    size = int(_lib.lib().vs_gated_linear_gradients_workspace(m, f, k, split, want_dx, want_dw_gate,
                                                                want_dw_up, aligned))
    ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    launch(x, "vs_gated_linear_gradients", DTYPES[x.dtype], ACTIVATIONS[activation], split, rows.data_ptr(),
           rows.stride(0), w_gate.data_ptr(), w_gate.stride(0), w_up.data_ptr(), w_up.stride(0), pre.data_ptr(),
           dhr.data_ptr(), dhr.stride(0), m, f, k, dx.data_ptr() if want_dx else None,
           dwg.data_ptr() if want_dw_gate else None, dwu.data_ptr() if want_dw_up else None, _opt(ws), size)
    return dx, dwg, dwu


def _gated_fake(x, w_gate, w_up, activation, save, split=False):
    _check_gated("veles::gated_linear", x, w_gate, w_up, activation)
    m, f = 1, w_gate.shape[0]
    for n in x.shape[:-1]:
        m = m * n
    return x.new_empty((*x.shape[:-1], f)), x.new_empty((m, f, 2) if save else (0,), dtype=torch.float32)


def _gated_setup(ctx, inputs, output):
    x, w_gate, w_up, activation, save, split = inputs
    if not save:
        raise RuntimeError("veles::gated_linear: gradients need the pre-activations (save=True)")
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, w_gate, w_up, output[1])
    ctx.activation, ctx.split = activation, split


def _gated_grad(ctx, dh, _):
    return *_gated_grads(ctx, torch.ops.veles.gated_linear_backward, dh), None, None, None


def _gated_grads(ctx, backward, dh):
    if dh is None:
        return None, None, None
    x, w_gate, w_up, pre = ctx.saved_tensors
    need = ctx.needs_input_grad
    grads = backward(x, w_gate, w_up, pre, dh, ctx.activation, *need[:3], ctx.split)
    return tuple(g if n else None for g, n in zip(grads, need))


class _Gated(torch.autograd.Function):
    """The op's autograd without the dispatcher."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation, split):
        h, pre = _gated_impl(x, w_gate, w_up, activation, True, split)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, w_gate, w_up, pre)
        ctx.activation, ctx.split = activation, split
        return h

    @staticmethod
    def backward(ctx, dh):
        # a graph of the gradients asks for second derivatives, which the op refuses by name
        op = torch.ops.veles.gated_linear_backward if torch.is_grad_enabled() else _gated_backward_impl
        return *_gated_grads(ctx, op, dh), None, None


torch.library.define("veles::gated_linear",
                     "(Tensor x, Tensor w_gate, Tensor w_up, str activation, bool save, bool split=False) -> "
                     "(Tensor, Tensor)")
torch.library.impl("veles::gated_linear", "default", _with_empty(_gated_impl))
torch.library.register_fake("veles::gated_linear", _gated_fake)
torch.library.register_autograd("veles::gated_linear", _gated_grad, setup_context=_gated_setup)
torch.library.define("veles::gated_linear_backward",
                     "(Tensor x, Tensor w_gate, Tensor w_up, Tensor pre, Tensor dh, str activation, bool want_dx, "
                     "bool want_dw_gate, bool? want_dw_up=None, bool split=False) -> (Tensor, Tensor, Tensor)")
torch.library.impl("veles::gated_linear_backward", "default", _gated_backward_impl)


def _gated_backward_fake(x, w_gate, w_up, pre, dh, activation, want_dx, want_dw_gate, want_dw_up=None, split=False):
    want_dw_up = want_dw_gate if want_dw_up is None else want_dw_up
    return (x.new_empty(x.shape if want_dx else (0,)), w_gate.new_empty(w_gate.shape if want_dw_gate else (0,)),
            w_up.new_empty(w_up.shape if want_dw_up else (0,)))


torch.library.register_fake("veles::gated_linear_backward", _gated_backward_fake)
_no_second_derivative("veles::gated_linear_backward")


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                 activation: str = "silu", split_gradients: bool = False) -> torch.Tensor:
    """act(x @ w_gate.T) * (x @ w_up.T): both products, the activation and the product of the two in one
    kernel, the first half of a gated feed-forward block.

    x: [..., k], weights [features, k], all float16 or all bfloat16; activation: silu, gelu (by the error
    function), relu or sigmoid.  Sums, activation and product are float32 and rounded once.  Differentiable
    in x and the weights; the float32 pairs (x @ w_gate.T, x @ w_up.T), 8 bytes per output, are kept for the
    backward pass.  There the gradients of the two products are rounded to x's type before they are multiplied,
    which adds about 0.4 of the result's own rounding to the error; in float16 they are lost below 6e-8 and
    infinite above 65504, so the loss has to be scaled.  split_gradients takes each as the sum of two numbers of x's
    type (to 2^-16 of it in bfloat16, to 2^-22 or 3e-8 in float16), so the result's own rounding is all that counts,
    for twice the multiplications of the backward pass (up to 2^19 features; on a CPU they are not rounded at all).  Up to 64 rows (generation) stream the weights once at memory speed."""
    save = records(x, w_gate, w_up)
    if plain_tensors(x, w_gate, w_up):
        if save:
            return _Gated.apply(x, w_gate, w_up, activation, split_gradients)
        return _gated_impl(x, w_gate, w_up, activation, False)[0]
    return torch.ops.veles.gated_linear(x, w_gate, w_up, activation, save, split_gradients)[0]
