"""Sequence operators over long behaviour histories, beside the pooling layers of din.py: layer
normalisation, a gated linear recurrence, and an encoder built of both.

    layer_norm(x, gamma, beta, epsilon, save_8bit)      LayerNormalization
    gated_recurrence(v, g, h0, lengths)                 GatedRecurrence
    gated_recurrence_step(v, g, state, out)             one event a session (serving)
    pack8 / unpack8                                     8-bit activation checkpoints (packing.py)
    SequenceEncoder                                     x + Dense(recurrence(norm(x))), stacked

The reference reads its behaviour sequences by pooling (din.py:18-47, staytime/layer.py:16-41) and
imports a LayerNormalization it does not hold (InteractingLayer.py:5); nothing in it depends on the
order of the events.  The recurrence does, at a cost linear in the length, and its state is all that
a served session has to keep.

    f_t = sigmoid(g_t)        h_t = f_t h_{t-1} + (1 - f_t) v_t

Rows are float32, bfloat16 or float16; gamma, beta, states and the parameters' gradients float32.
First derivatives in reverse mode only: second ones and forward mode (dual tensors) are refused.
"""
from __future__ import annotations

import functools

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, device_index, empty, empty_as, ptr, run_on
from .layers import Dense
from .packing import element_code, pack8, rows_of, scale_shape, unpack8  # noqa: F401
from .params import FlatBlock, grads_contiguous

MAX_WIDTH = 32768  # layer_norm's last dimension


def _first_order(backward):
    """backward as it is where no second derivative is asked for, and once_differentiable where one
    might be (create_graph), whose own work is left out otherwise."""
    once = once_differentiable(backward)
    return staticmethod(lambda ctx, *g: once(ctx, *g) if torch.is_grad_enabled() else backward(ctx, *g))


def _refuse_tangents(what, *tensors):
    """There is no forward-mode derivative: a dual tensor is refused, its tangent would be lost."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # no dual level is open (0.3 us a tensor less)
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative (jvp)")


# sizes that follow from a shape alone
@functools.lru_cache(maxsize=1024)
def _norm_workspace(R, D):
    return _lib.load().rs_layernorm_bwd_workspace_floats(R, D)


@functools.lru_cache(maxsize=1024)
def _rec_sizes(code, B, T, D):
    lib = _lib.load()
    return lib.rs_gated_rec_states_floats(code, B, T, D), lib.rs_gated_rec_workspace_floats(code, B, T, D)


# ============================================================================================
# layer normalisation
# ============================================================================================
def _check_norm(x, gamma, beta, epsilon):
    _refuse_tangents("layer_norm", x, gamma, beta)
    code = element_code(x, "layer_norm's input")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"layer_norm needs a last dimension of 1 to {MAX_WIDTH}, got shape "
                         f"{tuple(x.shape)}")
    D = x.shape[-1]
    for name, p in (("gamma", gamma), ("beta", beta)):
        if p.dtype is not torch.float32:
            raise TypeError(f"layer_norm: {name} must be float32, got {p.dtype}")
        if p.shape != (D,):
            raise ValueError(f"layer_norm: {name} {tuple(p.shape)} does not fit a last dimension of {D}")
    if not 1.2e-38 < epsilon < 3.4e38:
        raise ValueError(f"layer_norm: epsilon must be a positive float32 number, got {epsilon}")
    return code


def _norm_forward(x, gamma, beta, epsilon, code, stats, save_8bit, stream):
    x2 = rows_of(x)
    R, D = x2.shape
    y = empty_as(x)
    mean = codes = scales = None  # mean: [means | 1 / standard deviations]
    if stats:
        mean = empty((2, R))
    if save_8bit:
        codes, scales = empty_as(x, torch.int8), empty(scale_shape(x.shape))
    gamma, beta = gamma.contiguous(), beta.contiguous()  # (copies live until after the launch)
    call("rs_layernorm_fwd", stream, code, x2.data_ptr(), x2.stride(0), R, D, gamma.data_ptr(),
         beta.data_ptr(), epsilon, y.data_ptr(), D,
         ptr(mean), mean.data_ptr() + 4 * R if stats else None, ptr(codes), ptr(scales))
    return y, mean, codes, scales


def _norm_backward(dy, x, codes, scales, gamma, mean, code, dparams, accumulate, stream):
    """dx; dparams: [dgamma | dbeta], made here where it is None."""
    dy2 = rows_of(dy)
    R, D = dy2.shape
    x2 = rows_of(x) if x is not None else None
    dx = empty_as(dy)
    if dparams is None:
        dparams = empty((2, D))
    ws_n = _norm_workspace(R, D)
    ws = empty((ws_n,))
    gamma = gamma.contiguous()
    call("rs_layernorm_bwd", stream, code, dy2.data_ptr(), dy2.stride(0), ptr(x2),
         x2.stride(0) if x2 is not None else 0, ptr(codes), ptr(scales), R, D,
         gamma.data_ptr(), mean.data_ptr(), mean.data_ptr() + 4 * R, dx.data_ptr(), D,
         dparams.data_ptr(), dparams.data_ptr() + 4 * D, accumulate, ws.data_ptr(), ws_n)
    return dx, dparams


class _LayerNormFn(torch.autograd.Function):
    """in_place: add the parameters' gradients onto gamma.grad / beta.grad where these exist, and
    hand autograd None for them (the layers' way); otherwise return them."""

    @staticmethod
    def forward(ctx, x, gamma, beta, epsilon, code, save_8bit, in_place, index):
        y, mean, codes, scales = run_on(index, _norm_forward, x, gamma, beta, epsilon, code, True,
                                        save_8bit)
        ctx.save_for_backward(None if save_8bit else x, codes, scales, gamma, beta, mean)
        ctx.args = code, in_place, index
        return y

    @_first_order
    def backward(ctx, dy):
        x, codes, scales, gamma, beta, mean = ctx.saved_tensors
        code, in_place, index = ctx.args
        in_place = in_place and ctx.needs_input_grad[1] and ctx.needs_input_grad[2]
        block = grads_contiguous((gamma, beta)) if in_place else None
        dx, dparams = run_on(index, _norm_backward, dy, x, codes, scales, gamma, mean, code, block,
                             block is not None)
        dgamma, dbeta = dparams.unbind() if block is None else (None, None)
        return dx, dgamma, dbeta, None, None, None, None, None


def _norm(x, gamma, beta, epsilon, save_8bit, in_place):
    code = _check_norm(x, gamma, beta, epsilon)
    index = device_index(x, gamma, beta)
    train = torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad or beta.requires_grad)
    if _lib.CUSTOM_OPS["on"] and not (train and save_8bit):
        return torch.ops.ctr.layer_norm(x, gamma, beta, epsilon)[0]
    if train:
        return _LayerNormFn.apply(x, gamma, beta, epsilon, code, save_8bit, in_place, index)
    return run_on(index, _norm_forward, x, gamma, beta, epsilon, code, False, False)[0]


def layer_norm(x, gamma, beta, epsilon=1e-5, save_8bit=False):
    """(x - mean) / sqrt(var + epsilon) * gamma + beta over the last dimension (1 to 32768) of x
    (float32 / bfloat16 / float16, any leading shape and strides); gamma and beta float32.
    save_8bit: keep x for the backward in 8 bits (packing.py) instead of as it is; y, mean and
    variance are those of x itself, and so is the sum of dy; the normalised rows that dx and
    dgamma are computed with are those of the kept values.
    Sums are float32: a row whose squared deviations sum past its range (deviations of 1e18 or
    so) gives beta."""
    return _norm(x, gamma, beta, float(epsilon), bool(save_8bit), False)


class LayerNormalization(nn.Module):
    """layer_normalization.LayerNormalization (InteractingLayer.py:5,28) as a layer of its own:
    gamma ones, beta zeros, built on the first call from the input's last dimension."""

    def __init__(self, epsilon=1e-5, save_8bit=False, device=None, name=None):
        super().__init__()
        self.epsilon = float(epsilon)
        self.save_8bit = bool(save_8bit)
        self._device = device
        self.built = False
        self.name = name

    def build(self, input_shape, device=None):
        D = int(input_shape[-1])
        self.gamma, self.beta = FlatBlock([(D,), (D,)], device or self._device or
                                          torch.device("cuda")).params()
        with torch.no_grad():
            self.gamma.fill_(1.0)
        self.input_dim = D
        self.built = True

    def forward(self, x):
        if not self.built:
            self.build(tuple(x.shape), device=x.device)
        return _norm(x, self.gamma, self.beta, self.epsilon, self.save_8bit, True)


# ============================================================================================
# gated linear recurrence
# ============================================================================================
MAX_STEP_STRIDE = 2 ** 23  # elements between two steps (and of a step) that the kernels index


def _strided(t):
    """t [B, T, D] as the kernels read it, and its batch and step strides: in place with unit stride
    along D and steps not too far apart, a contiguous copy otherwise.  A single step has no next one:
    whatever its stride says (a view of time-major rows may say anything) is not passed on."""
    sb, st, sc = t.stride()
    if t.shape[1] <= 1:
        st = 0
    if (sc != 1 and t.shape[2] != 1) or st >= MAX_STEP_STRIDE:
        t = t.contiguous()
        sb, st, _ = t.stride()
    return t, sb, st


def _halves(v, g):
    """The value and gate rows: (v, g) as they are, or the halves of v's last dimension."""
    if g is not None:
        return v, g
    D = v.shape[-1] // 2
    return v[..., :D], v[..., D:]


def _check_rec(v, g, dims, what):
    _refuse_tangents(what, v, g)
    if v.dim() != dims:
        raise ValueError(f"{what} takes rank-{dims} values, got shape {tuple(v.shape)}")
    code = element_code(v, f"{what}'s values")
    if g is None:
        if v.shape[-1] < 2 or v.shape[-1] % 2:
            raise ValueError(f"{what} without g takes [values | gates] in one last dimension, which "
                             f"must be even and not 0, got {v.shape[-1]}")
    else:
        if g.dtype != v.dtype:
            raise TypeError(f"{what}: values and gates differ in type: {v.dtype} and {g.dtype}")
        if g.shape != v.shape:
            raise ValueError(f"{what}: values {tuple(v.shape)} and gates {tuple(g.shape)} differ in shape")
        if v.shape[-1] < 1:
            raise ValueError(f"{what} needs a last dimension of at least 1, got shape {tuple(v.shape)}")
    if v.shape[-1] >= MAX_STEP_STRIDE:
        raise ValueError(f"{what}: a last dimension of {v.shape[-1]} is not supported")
    return code


def _any_grad(*tensors):
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _check_state(state, shape, what):
    if state is None:
        return
    _refuse_tangents(what, state)
    if state.dtype is not torch.float32:
        raise TypeError(f"{what} must be float32, got {state.dtype}")
    if state.shape != shape:
        raise ValueError(f"{what} must be {shape}, got {tuple(state.shape)}")


def _rec_forward(v, g, h0, lengths, code, keep, stream):
    v, g = _halves(v, g)
    B, T, D = v.shape
    v, v_sb, v_st = _strided(v)
    g, g_sb, g_st = _strided(g)
    n_states, n_ws = _rec_sizes(code, B, T, D)
    h = empty_as(v)
    last = empty((B, D))
    states = empty((n_states,)) if keep and n_states else None
    ws = empty((n_ws,)) if n_ws else None
    call("rs_gated_rec_fwd", stream, code, v.data_ptr(), v_sb, v_st, g.data_ptr(), g_sb, g_st, B, T, D,
         ptr(lengths), ptr(h0), h.data_ptr(), last.data_ptr(), ptr(states), ptr(ws), n_ws)
    return h, last, states


def _rec_backward(v, g, h0, lengths, states, dh, dlast, code, want_h0, stream):
    """(dv, dg, dh0); with g None dv is the gradient of the joint rows and dg None."""
    joint = g is None
    dvg = empty_as(v)
    dv, dg = _halves(dvg, None if joint else empty_as(v))
    v, g = _halves(v, g)
    B, T, D = v.shape
    v, v_sb, v_st = _strided(v)
    g, g_sb, g_st = _strided(g)
    d_sb, d_st, _ = dv.stride()
    dh_sb = dh_st = 0
    if dh is not None:
        dh, dh_sb, dh_st = _strided(dh)
    if dlast is not None:
        dlast = dlast.contiguous()
    dh0 = empty((B, D)) if want_h0 else None
    n_ws = _rec_sizes(code, B, T, D)[1]
    ws = empty((n_ws,)) if n_ws else None
    call("rs_gated_rec_bwd", stream, code, v.data_ptr(), v_sb, v_st, g.data_ptr(), g_sb, g_st, B, T, D,
         ptr(lengths), ptr(h0), ptr(states), ptr(dh), dh_sb, dh_st, ptr(dlast), dv.data_ptr(), d_sb, d_st,
         dg.data_ptr(), d_sb, d_st, ptr(dh0), ptr(ws), n_ws)
    return dvg, None if joint else dg, dh0


class _RecurrenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, v, g, h0, lengths, code, index):
        ctx.set_materialize_grads(False)
        h, last, states = run_on(index, _rec_forward, v, g, h0, lengths, code, True)
        ctx.save_for_backward(v, g, h0, lengths, states)
        ctx.args = code, index
        return h, last

    @_first_order
    def backward(ctx, dh, dlast):
        v, g, h0, lengths, states = ctx.saved_tensors
        if dh is None and dlast is None:
            return None, None, None, None, None, None
        code, index = ctx.args
        return (*run_on(index, _rec_backward, v, g, h0, lengths, states, dh, dlast, code,
                        ctx.needs_input_grad[2]), None, None, None)


def _check_lengths(lengths, B, T):
    if lengths is None:
        return None
    if lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"lengths must be int32 or int64, got {lengths.dtype}")
    if tuple(lengths.shape) != (B,):
        raise ValueError(f"lengths must be ({B},), got {tuple(lengths.shape)}")
    if lengths.dtype == torch.int64:  # into 0..T before the narrower type could wrap
        lengths = lengths.clamp(0, T).to(torch.int32)
    return lengths.contiguous()


def gated_recurrence(v, g=None, h0=None, lengths=None):
    """h_t = f_t h_{t-1} + (1 - f_t) v_t with f_t = sigmoid(g_t), over v, g [B, T, D]; returns
    (h [B, T, D] in the rows' type, the state after the last step [B, D] float32).

    g None: v is [B, T, 2 D], values and gates side by side, as one Dense(2 D) gives them.
    h0 [B, D] float32: the state before the first step (default zeros).
    lengths int32 / int64 [B]: steps from lengths[b] on are not part of the sequence (values are
    taken into 0..T): whatever v and g hold there, h is zero, no gradient flows, and the returned
    state is that after lengths[b] steps (h0 for an empty sequence).
    v, g: float32 / bfloat16 / float16, any strides (unit along D is read in place).
    The smaller of f and 1 - f is held to its own digits, to some 2^-21 of itself for float32 rows; for
    16-bit rows the exponential's argument is rounded too, |g| 2^-24 more, which h does not show but
    the float32 state and h0's gradient carry.  Values and states have to be finite: an infinity
    gives NaN in its channel from the same step on or a later one, where the formula would stay infinite."""
    code = _check_rec(v, g, 3, "gated_recurrence")
    B, T, D = v.shape if g is not None else (*v.shape[:2], v.shape[2] // 2)
    _check_state(h0, (B, D), "gated_recurrence: h0")
    index = device_index(v, g, h0, lengths)
    lengths = _check_lengths(lengths, B, T)
    if _lib.CUSTOM_OPS["on"]:
        return tuple(torch.ops.ctr.gated_recurrence(v, g, h0, lengths)[:2])
    if h0 is not None:
        h0 = h0.contiguous()
    if torch.is_grad_enabled() and _any_grad(v, g, h0):
        return _RecurrenceFn.apply(v, g, h0, lengths, code, index)
    return run_on(index, _rec_forward, v, g, h0, lengths, code, False)[:2]


def gated_recurrence_step(v, g=None, state=None, out=None):
    """One step for B sessions: v, g [B, D] (g None: v [B, 2 D]), state [B, D] float32 (None:
    zeros) -> (h [B, D] in the rows' type, the new state [B, D] float32).  out: where the new
    state goes (a contiguous float32 [B, D]; may be `state` itself, which is then updated in
    place; overlaps no other argument).  Under autograd use gated_recurrence, of which this is the case T = 1."""
    code = _check_rec(v, g, 2, "gated_recurrence_step")
    B, D = v.shape if g is not None else (v.shape[0], v.shape[1] // 2)
    _check_state(state, (B, D), "gated_recurrence_step: state")
    _check_state(out, (B, D), "gated_recurrence_step: out")
    if out is not None and not out.is_contiguous():
        raise ValueError("gated_recurrence_step: out must be contiguous")
    if torch.is_grad_enabled() and _any_grad(v, g, state, out):
        raise RuntimeError("gated_recurrence_step has no backward: call it under torch.no_grad(), or "
                           "gated_recurrence with one step")
    index = device_index(v, g, state, out)
    if _lib.CUSTOM_OPS["on"]:
        h, new = torch.ops.ctr.gated_recurrence_step(v, g, state)
        return h, new if out is None else out.copy_(new)
    if out is not None:
        _check_out(out, v, g, state)
    return run_on(index, _rec_step, v, g, state, out, B, D, code)


def _check_out(out, v, g, state):
    """The step writes out while other threads still read: it may be the state itself (every element
    is read and written by one thread), but not overlap anything otherwise."""
    begin = out.data_ptr()
    end = begin + 4 * out.numel()
    for name, t in (("the values", v), ("the gates", g), ("the state", state)):
        if t is None or t is out or not t.numel():
            continue
        at = t.data_ptr()
        if at >= end or (name == "the state" and (at == begin or not t.is_contiguous())):  # (copied first)
            continue
        if begin < at + ((t.shape[0] - 1) * t.stride(0) + (t.shape[1] - 1) * t.stride(1) + 1) * t.element_size():
            raise ValueError(f"gated_recurrence_step: out overlaps {name}")


def _rec_step(v, g, state, out, B, D, code, stream):
    v, g = _halves(v, g)
    if D > 1:
        v, g = (t if t.stride(1) == 1 else t.contiguous() for t in (v, g))
    if state is not None:
        state = state.contiguous()
    h = empty_as(v)
    if out is None:
        out = empty((B, D))
    call("rs_gated_rec_step", stream, code, v.data_ptr(), v.stride(0), g.data_ptr(), g.stride(0), B, D,
         ptr(state), h.data_ptr(), out.data_ptr())
    return h, out


class GatedRecurrence(nn.Module):
    """[v | g] = Dense(2 units)(x), then gated_recurrence over the steps of x [B, T, E]:
    layer(x, lengths, state) -> (h [B, T, units], the state after the last step [B, units]).
    forget_bias: initial bias of the gates (2: memories of about 8 steps).  save_8bit: keep the
    projection's input for its backward in 8 bits."""

    def __init__(self, units, forget_bias=2.0, seed=0, save_8bit=False, device=None, name=None):
        super().__init__()
        self.units = int(units)
        if self.units < 1:
            raise ValueError(f"GatedRecurrence needs at least one unit, got {units}")
        self.forget_bias = float(forget_bias)
        self.projection = Dense(2 * self.units, seed=seed, device=device, save_8bit=save_8bit)
        self.built = False
        self.name = name

    def build(self, input_shape, device=None):
        if not self.projection.built:
            self.projection.build(input_shape, device=device)
            with torch.no_grad():
                self.projection.bias[self.units:].fill_(self.forget_bias)
        self.built = True

    def forward(self, x, lengths=None, state=None):
        if x.dim() != 3:
            raise ValueError('The rank of input of GatedRecurrence must be 3, but now is %d' % x.dim())
        if not self.built:
            self.build(tuple(x.shape), device=x.device)
        return gated_recurrence(self.projection(x), None, state, lengths)

    @torch.no_grad()
    def step(self, x, state=None, out=None):
        """One event a session: x [B, E] -> (h [B, units], new state)."""
        if x.dim() != 2:
            raise ValueError('The rank of input of GatedRecurrence.step must be 2, but now is %d' % x.dim())
        if not self.built:
            self.build(tuple(x.shape), device=x.device)
        return gated_recurrence_step(self.projection(x), None, state, out)


class SequenceEncoder(nn.Module):
    """`depth` residual blocks x + Dense(E)(recurrence(norm(x))) over a history x [B, T, E], with a
    last normalisation: encoder(x, lengths, states) -> (y [B, T, E], states [depth, B, units]).
    Rows behind lengths[b] may hold anything, NaN included; y and x's gradient are zero there.
    states: those an earlier call returned for the sessions (the history read so far); `step` goes
    on from there with one event a session.  save_8bit: the normalisations and projections keep
    their inputs for the backward in 8 bits."""

    def __init__(self, units, depth=1, forget_bias=2.0, epsilon=1e-5, seed=0, save_8bit=False,
                 device=None, name=None):
        super().__init__()
        if depth < 1:
            raise ValueError(f"SequenceEncoder needs at least one block, got depth {depth}")
        self.units, self.depth = int(units), int(depth)
        self.norms = nn.ModuleList(LayerNormalization(epsilon, save_8bit, device) for _ in range(depth))
        self.recurrences = nn.ModuleList(
            GatedRecurrence(units, forget_bias, seed + 2 * k, save_8bit, device) for k in range(depth))
        self._out = [dict(seed=seed + 2 * k + 1, device=device, save_8bit=save_8bit) for k in range(depth)]
        self.final = LayerNormalization(epsilon, save_8bit, device)
        self.built = False
        self.name = name

    def build(self, input_shape, device=None):
        E = int(input_shape[-1])
        self.outputs = nn.ModuleList()
        for k in range(self.depth):
            self.norms[k].build((E,), device)
            self.recurrences[k].build((E,), device)
            out = Dense(E, **self._out[k])
            out.build((self.units,), device)
            self.outputs.append(out)
        self.final.build((E,), device)
        self.built = True

    def _check(self, x, states, rank, what):
        if x.dim() != rank:
            raise ValueError(f'The rank of input of {what} must be {rank}, but now is {x.dim()}')
        want = (self.depth, x.shape[0], self.units)
        if states is not None and tuple(states.shape) != want:
            raise ValueError(f"{what}: states must be {want}, got {tuple(states.shape)}")
        if not self.built:
            self.build(tuple(x.shape), device=x.device)

    def forward(self, x, lengths=None, states=None):
        self._check(x, states, 3, "SequenceEncoder")
        x = x.float()
        B, T = x.shape[:2]
        keep = None
        if lengths is not None:
            lengths = _check_lengths(lengths, B, T)
            keep = (torch.arange(T, device=x.device) < lengths.unsqueeze(1)).unsqueeze(2)
            x = x.masked_fill(~keep, 0.0)
        last = []
        for k in range(self.depth):
            h, s = self.recurrences[k](self.norms[k](x), lengths, None if states is None else states[k])
            x = x + self.outputs[k](h)
            last.append(s)
        y = self.final(x)
        return (y if keep is None else y.masked_fill(~keep, 0.0)), torch.stack(last)

    @torch.no_grad()
    def step(self, x, states=None):
        """One event a session: x [B, E] -> (y [B, E], new states [depth, B, units])."""
        self._check(x, states, 2, "SequenceEncoder.step")
        x = x.float()
        new = torch.empty(self.depth, x.shape[0], self.units, device=x.device, dtype=torch.float32)
        for k in range(self.depth):
            h, _ = self.recurrences[k].step(self.norms[k](x), None if states is None else states[k],
                                            new[k])
            x = x + self.outputs[k](h)
        return self.final(x), new
