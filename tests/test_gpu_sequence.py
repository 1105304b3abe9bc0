"""GPU: layer normalisation, the gated linear recurrence and 8-bit checkpoints against their
definitions in 64 bits on the CPU.

Tolerances.  u = 2^-24 is the half step of fp32, half(t) that of the rows' type.  An output is
rounded once: half(t) |value|.  Below fp16's normal range (2^-14) the step is fixed: 2^-25 absolute.
  * layer norm: a thread adds at most 32 of a row's elements, then 10 levels of a tree, so a sum is
    off by at most 48 u of the sum of magnitudes; with the few operations around it 64 u of the
    magnitudes that enter an output bounds its fp32 error.
  * parameter gradients: at the sizes here a thread adds at most 160 rows one after the other,
    the rest is trees; with the error of the normalised value 256 u of the sum of magnitudes.
  * recurrence: the error of a state obeys the recurrence itself, e_t = f_t e_{t-1} + what step t
    adds: 2 u for each of its roundings and 4 u of its input for the gate (exp and reciprocal),
    taken as 16 u of the magnitudes, which also covers joining partial results in another order
    (each join rounds values no larger than the sum of the magnitudes of the state's terms, and a
    step lies under at most 16 joins).
"""
from __future__ import annotations

import pytest
import torch

from recommendsystem_amd import (Dense, GatedRecurrence, LayerNormalization, SequenceEncoder,
                                 gated_recurrence, gated_recurrence_step, layer_norm, pack8, unpack8)

from _rec_forms import FORMS

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
names = lambda t: str(t).split(".")[-1]  # noqa: E731


def near(got, ref, bound, what):
    """|got - ref| <= the rounding of got's type + bound (both of ref's shape)."""
    assert tuple(got.shape) == tuple(ref.shape), (what, got.shape, ref.shape)
    g = got.detach().double().cpu()
    tol = HALF[got.dtype] * ref.abs() + bound * (1 + HALF[got.dtype]) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    bad = (g - ref).abs() - tol
    if bad.numel() and not bool((bad <= 0).all()):
        i = int(torch.nan_to_num(bad, nan=float("inf")).argmax())
        raise AssertionError(f"{what}: {int((~(bad <= 0)).sum())} of {bad.numel()} off, worst got "
                             f"{g.flatten()[i]:.9g}, want {ref.flatten()[i]:.9g} +- {tol.flatten()[i]:.3g} at {i}")


def rnd(*shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(*shape, device=DEV) * std + mean).to(dtype)


# ============================================================================================
# 8-bit form
# ============================================================================================
def ref_pack(x):
    """codes (float64) and scales from the definition; x on the CPU, [R, D] float64."""
    R, D = x.shape
    codes, scales = torch.zeros_like(x), []
    for lo in range(0, D, 128):
        part = x[:, lo:lo + 128]
        top = part.abs().amax(1, keepdim=True)
        s = (top / 127).float().double()
        s = torch.where(top < 2.0 ** -100, torch.zeros_like(s), s)
        codes[:, lo:lo + 128] = torch.where(s > 0, torch.round(part / torch.where(s > 0, s, torch.ones_like(s))),
                                            torch.zeros_like(part))
        scales.append(s)
    return codes, torch.cat(scales, 1)


def unpacked(codes, scales):
    return codes * scales.repeat_interleave(128, 1)[:, :codes.shape[1]]


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("R,D", [(1, 1), (3, 7), (5, 64), (2, 127), (9, 128), (4, 129), (33, 200), (7, 1456),
                                 (1, 5003), (300, 16)])
def test_pack8(R, D, dtype):
    x = rnd(R, D, dtype=dtype) * (torch.rand(R, 1, device=DEV) * 30).to(dtype)
    codes, scales = pack8(x)
    want, ws = ref_pack(x.double().cpu())
    assert torch.equal(scales.double().cpu(), ws)
    assert torch.equal(codes.double().cpu(), want)
    for t in TYPES:
        y = unpack8(codes, scales, t)
        near(y, unpacked(want, ws), 0.0, f"unpack8 to {t}")


def test_pack8_ties_zeros_and_strides():
    # scale 1: whole and half numbers; scale 3 (not a power of two): true ties at 1.5 (2 k + 1)
    rows = [torch.arange(-127, 128, 2).double() / 2, (torch.arange(128).double() - 64) * 1.5]
    rows[0][0], rows[1][0] = 127.0, 381.0
    x = torch.stack([rows[0][:128], rows[1]]).to(DEV)
    for t in (torch.float32, torch.float16):
        codes, scales = pack8(x.to(t))
        want, ws = ref_pack(x.cpu())
        assert torch.equal(codes.double().cpu(), want) and torch.equal(scales.double().cpu(), ws)
    z = torch.zeros(3, 130, device=DEV)
    z[1, :128] = 1e-31
    z[2] = 2.0 ** -100
    codes, scales = pack8(z)
    assert not codes[:2].any() and not scales[:2].any()
    assert torch.equal(codes[2], torch.full_like(codes[2], 127))
    # columns of a wider buffer, transposed rows, an expanded row, higher ranks, nothing at all
    wide = rnd(6, 300)
    for x in (wide[:, 3:133], wide.t(), wide[:1].expand(5, 300), wide.view(2, 3, 300)[:, 1:], wide[:0]):
        codes, scales = pack8(x)
        assert codes.shape == x.shape
        flat = x.reshape(-1, x.shape[-1])
        want, ws = ref_pack(flat.double().cpu())
        assert torch.equal(codes.reshape(flat.shape).double().cpu(), want)
        assert torch.equal(unpack8(codes, scales).reshape(flat.shape).double().cpu(),
                           unpacked(want, ws).float().double())


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_pack8_not_finite(dtype):
    x = torch.ones(3, 256, device=DEV, dtype=dtype)
    x[0, 5], x[1, 130], x[2, 255] = float("nan"), float("inf"), float("-inf")
    y = unpack8(*pack8(x), dtype)
    bad = torch.zeros(3, 256, dtype=torch.bool)
    bad[0, :128] = bad[1, 128:] = bad[2, 128:] = True
    assert torch.equal(y.isnan().cpu(), bad)
    assert torch.equal(y[~y.isnan()], x[:1].new_ones(1).expand(int((~bad).sum())))


# ============================================================================================
# layer normalisation
# ============================================================================================
def ref_norm(x, gamma, beta, eps, dy=None, at=None):
    """(value, bound) pairs of y and, with dy, dx, dgamma, dbeta; float64 on the CPU."""
    x, gamma, beta = x.double().cpu(), gamma.detach().double().cpu(), beta.detach().double().cpu()
    D = x.shape[1]
    mean = x.mean(1, keepdim=True)
    var = (x - mean).pow(2).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * r
    out = [(xh * gamma + beta, 64 * U * ((xh.abs() + 1) * gamma.abs() + beta.abs()))]
    if dy is None:
        return out
    dy = dy.double().cpu()
    slack = torch.zeros_like(r)
    if at is not None:  # the kept values against the row's own mean, which fp32 holds to u |mean|
        xh = (at - mean) * r
        slack = 2 * U * mean.abs() * r
    w = dy * gamma
    c1, c2 = w.mean(1, keepdim=True), (w * xh).mean(1, keepdim=True)
    mag = w.abs() + w.abs().mean(1, keepdim=True) + (xh.abs() + 1) * ((w * xh).abs().mean(1, keepdim=True)
                                                                   + w.abs().mean(1, keepdim=True))
    # a shift of xh by slack moves c2 by slack mean|w| and xh c2 by slack (|c2| + |xh| mean|w|)
    sl = slack * (c2.abs() + xh.abs() * w.abs().mean(1, keepdim=True))
    out.append((r * (w - c1 - xh * c2), r * (64 * U * mag + sl)))
    out.append(((dy * xh).sum(0), 256 * U * (dy.abs() * (xh.abs() + 1)).sum(0) + (dy.abs() * slack).sum(0)))
    out.append((dy.sum(0), 256 * U * dy.abs().sum(0)))
    return out


NORM_SHAPES = [(1, 1), (3, 1), (1, 2), (5, 3), (7, 8), (3, 16), (130, 31), (65, 32), (64, 33), (9, 64), (17, 100),
               (33, 128), (6, 129), (5, 255), (4, 256), (3, 257), (1025, 264), (2, 512), (5, 513), (9, 1000),
               (3, 1024), (2, 1025), (3, 1456), (2, 2048), (3, 2049), (5, 4096), (2, 5003), (1, 8192),
               (2, 8193), (2, 12000), (3, 16385), (1, 32767), (2, 32768), (5000, 20)]


@pytest.mark.parametrize("save_8bit", [False, True], ids=["", "8bit"])
@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("R,D", NORM_SHAPES)
def test_layer_norm(R, D, dtype, save_8bit):
    x = (rnd(R, D) * (0.5 + torch.rand(R, 1, device=DEV)) + rnd(R, 1)).to(dtype).requires_grad_()
    gamma, beta = rnd(D, mean=1.0, std=0.2).requires_grad_(), rnd(D).requires_grad_()
    dy = rnd(R, D, dtype=dtype)
    y = layer_norm(x, gamma, beta, 1e-5, save_8bit)
    grads = torch.autograd.grad(y, (x, gamma, beta), dy)
    at = unpacked(*ref_pack(x.detach().double().cpu())) if save_8bit else None
    for got, (want, bound), what in zip((y, *grads), ref_norm(x.detach(), gamma, beta, 1e-5, dy, at),
                                        ("y", "dx", "dgamma", "dbeta")):
        near(got, want, bound, what)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, gamma, beta, 1e-5), y)
    again = torch.autograd.grad(layer_norm(x, gamma, beta, 1e-5, save_8bit), (x, gamma, beta), dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_layer_norm_offset_constant_and_not_finite():
    # an offset 10^4 times the spread costs no digits; a constant row gives beta and no gradient
    x = rnd(6, 300) + 1e4
    x[4] = 12345.678
    gamma, beta = rnd(300, mean=1.0, std=0.1), rnd(300)
    dy = rnd(6, 300)
    xr = x.clone().requires_grad_()
    y = layer_norm(xr, gamma, beta, 1e-5)
    dx, = torch.autograd.grad(y, xr, dy)
    want = ref_norm(x, gamma, beta, 1e-5, dy)
    near(y, *want[0], "y")
    near(dx, *want[1], "dx")
    assert torch.equal(y[4], beta)
    for D in (1, 7, 300, 5000, 20000):  # also where epsilon gives no slack at all
        x, beta = torch.full((2, D), 0.1, device=DEV), rnd(D)
        assert torch.equal(layer_norm(x, rnd(D), beta, 1e-14), beta.expand(2, D))
    # one row's NaN or infinity stays in that row
    x = rnd(5, 700)
    x[1, 3], x[3, 699] = float("nan"), float("inf")
    y = layer_norm(x, rnd(700), rnd(700))
    assert torch.equal(y.isnan().all(1).cpu(), torch.tensor([False, True, False, True, False]))
    assert not y[[0, 2, 4]].isnan().any()


@pytest.mark.parametrize("save_8bit", [False, True], ids=["", "8bit"])
@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("D", [2, 40, 300, 1024, 8192, 16385, 32768])
@pytest.mark.parametrize("at", [0, -1])
def test_layer_norm_outlier(at, D, dtype, save_8bit):
    """One channel far above the others, as residual streams have them, the first one or the last: it
    takes no digits from the others.  A sum is off by 48 u of its terms' magnitudes, the mean so by 48 u
    of the mean |deviation|, which is far below the standard deviation here: 64 u (|xh| + mean |xh|)."""
    x = rnd(3, D)
    x[:, at] = 3e4 if dtype is torch.float16 else 1e6
    x = x.to(dtype).requires_grad_()
    gamma, beta = rnd(D, mean=1.0, std=0.2).requires_grad_(), rnd(D).requires_grad_()
    dy = rnd(3, D, dtype=dtype)
    y = layer_norm(x, gamma, beta, 1e-5, save_8bit)
    grads = torch.autograd.grad(y, (x, gamma, beta), dy)
    kept = unpacked(*ref_pack(x.detach().double().cpu())) if save_8bit else None
    want = ref_norm(x.detach(), gamma, beta, 1e-5, dy, kept)
    xd, gd = x.detach().double().cpu(), gamma.detach().double().cpu()
    dev = xd - xd.mean(1, keepdim=True)
    xh = dev.abs() / torch.sqrt(dev.pow(2).mean(1, keepdim=True) + 1e-5)
    want[0] = want[0][0], 64 * U * (xh + xh.mean(1, keepdim=True)) * gd.abs() + 4 * U * beta.detach().double().cpu().abs()
    for got, (w, bound), what in zip((y, *grads), want, ("y", "dx", "dgamma", "dbeta")):
        near(got, w, bound, what)


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_layer_norm_of_one_column(dtype):
    """y is beta whatever x is, so x's gradient is zero, to the last bit.  Kept in 8 bits x comes back
    within 2 u |x| (the scale's rounding and the product's), d, and dx = -w d^2 / sd^3."""
    x, dy = rnd(912, 1, dtype=dtype).requires_grad_(), rnd(912, 1, dtype=dtype)
    gamma, beta = rnd(1, mean=1.0).requires_grad_(), rnd(1).requires_grad_()
    for save_8bit in (False, True):
        y = layer_norm(x, gamma, beta, 1e-5, save_8bit)
        assert torch.equal(y, beta.to(dtype).expand(912, 1))
        dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), dy)
        d = 2 * U * x.detach().double().abs() * (save_8bit * 1.01)
        w = (dy.double() * gamma.detach().double()).abs()
        assert bool((dx.double().abs() <= w * d * d * 1e-5 ** -1.5).all())
        assert float(dgamma.detach()) <= float((dy.double().abs() * d).sum()) * 1e-5 ** -0.5
        near(dbeta, dy.double().cpu().sum(0), 256 * U * dy.double().cpu().abs().sum(0), "dbeta")


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_layer_norm_kept_values_are_those_of_unpack8(dtype):
    """In one column all that is left of the kept value is its rounding: the gradient sees the number that
    unpack8 gives, not a product carried on without rounding."""
    x, dy = rnd(900, 1, dtype=dtype).requires_grad_(), rnd(900, 1, dtype=dtype)
    gamma = rnd(1, mean=1.0).requires_grad_()
    dgamma, = torch.autograd.grad(layer_norm(x, gamma, rnd(1), 1e-5, True), gamma, dy)
    d = unpack8(*pack8(x)).double().cpu() - x.detach().double().cpu()
    terms = dy.double().cpu() * d * 1e-5 ** -0.5
    # (16-bit values mostly come back whole: fl(fl(m / 127) 127) = m for all 8-bit m, and all but 7 11-bit ones)
    assert bool(d.any()) or dtype is not torch.float32
    near(dgamma, terms.sum(0), 256 * U * terms.abs().sum(0), "dgamma")


def test_layer_norm_strides_ranks_and_empty():
    gamma, beta = rnd(40, mean=1.0).requires_grad_(), rnd(40).requires_grad_()
    wide = rnd(12, 100)
    for x in (wide[:, 5:45], wide.view(3, 4, 100)[:, :, 60:], wide[:40 // 4, :40].t().reshape(10, 40),
              wide[:1, :40].expand(7, 40), rnd(40, 9).t(), rnd(40), wide.view(3, 4, 100)[:, 1:3, :40]):
        x = x.detach().requires_grad_()
        dy = rnd(40).expand(x.shape)  # stride 0 rows
        y = layer_norm(x, gamma, beta)
        got = (y, *torch.autograd.grad(y, (x, gamma, beta), dy))
        want = ref_norm(x.detach().reshape(-1, 40), gamma, beta, 1e-5, dy.reshape(-1, 40))
        for g, (w, b), shape in zip(got, want, (x.shape, x.shape, (40,), (40,))):
            near(g, w.reshape(shape), b.reshape(shape), f"strides {x.stride()}")
    x = rnd(0, 3, 40).requires_grad_()
    dx, dg, db = torch.autograd.grad(layer_norm(x, gamma, beta), (x, gamma, beta), rnd(0, 3, 40))
    assert dx.shape == x.shape and not dg.any() and not db.any()


def test_layer_norm_parameters_of_any_stride_and_frozen():
    """gamma and beta as columns of one matrix; a frozen beta's gradient buffer is left alone."""
    p = rnd(40, 2)
    x, dy = rnd(6, 40), rnd(6, 40)
    gamma, beta = p[:, 0].requires_grad_(), p[:, 1].requires_grad_()
    y = layer_norm(x, gamma, beta)
    got = (y, *torch.autograd.grad(y, (gamma, beta), dy))
    want = ref_norm(x, gamma, beta, 1e-5, dy)
    for a, (w, b) in zip(got, (want[0], want[2], want[3])):
        near(a, w, b, "strided parameters")
    ln = LayerNormalization()
    ln.build((40,))
    ln.beta.requires_grad_(False)
    ln.beta.grad.fill_(7.0)
    ln(x).backward(dy)
    near(ln.gamma.grad, *ref_norm(x, ln.gamma, ln.beta, 1e-5, dy)[2], "dgamma")
    assert bool((ln.beta.grad == 7.0).all())


def test_layer_norm_differences():
    """The gradient against central differences of the 64-bit loss of the fp32 output: with a step
    h = 2^-5 the quotient is off by h^2/6 of a third derivative (of order 1 a unit direction) and by
    the output's rounding over h: 1e-3 of the gradient's norm covers both."""
    x, gamma, beta, dy = rnd(4, 60), rnd(60, mean=1.0, std=0.2), rnd(60), rnd(4, 60)
    xr, gr, br = (t.clone().requires_grad_() for t in (x, gamma, beta))
    grads = torch.autograd.grad(layer_norm(xr, gr, br), (xr, gr, br), dy)
    loss = lambda a, b, c: float((layer_norm(a, b, c).double() * dy.double()).sum())  # noqa: E731
    for k, t in enumerate((x, gamma, beta)):
        d = rnd(*t.shape)
        d /= d.norm()
        h = 2.0 ** -5
        args = lambda s: [p + s * d if i == k else p for i, p in enumerate((x, gamma, beta))]  # noqa: E731
        diff = (loss(*args(h)) - loss(*args(-h))) / (2 * h)
        assert abs(diff - float((grads[k] * d).double().sum())) <= 1e-3 * float(grads[k].norm())


def test_layer_normalization_layer():
    ln = LayerNormalization(epsilon=1e-3)
    x = rnd(5, 6, 48).requires_grad_()
    y = ln(x)
    dy = rnd(5, 6, 48)
    y.backward(dy)
    want = ref_norm(x.detach().reshape(-1, 48), ln.gamma, ln.beta, 1e-3, dy.reshape(-1, 48))
    near(ln.gamma.grad, *want[2], "dgamma")
    near(ln.beta.grad, *want[3], "dbeta")
    before = ln.gamma.grad.clone()
    ln(x).backward(dy)          # accumulates in place, as the other layers do
    near(ln.gamma.grad, want[2][0] + before.double().cpu(), 2 * want[2][1], "accumulated")


# ============================================================================================
# gated linear recurrence
# ============================================================================================
def ref_rec(v, g, h0, lengths, dh=None, dlast=None):
    """(value, bound) pairs of h, last and, with dh, dv, dg, dh0; float64 on the CPU."""
    hf = HALF[v.dtype]
    v, g = v.double().cpu(), g.double().cpu()
    B, T, D = v.shape
    n = lengths.cpu().long().clamp(0, T) if lengths is not None else torch.full((B,), T)
    live = (torch.arange(T).unsqueeze(0) < n.unsqueeze(1)).unsqueeze(2)
    v = torch.where(live, v, torch.zeros(()).double())
    i = torch.where(live, torch.sigmoid(-g), torch.zeros(()).double())
    f = torch.where(live, torch.sigmoid(g), torch.ones(()).double())
    s = h0.double().cpu() if h0 is not None else torch.zeros(B, D).double()
    e, top = torch.zeros(B, D).double(), s.abs()
    hs, es = [s], [e]
    for t in range(T):
        new = s + i[:, t] * (v[:, t] - s)
        # (top: the sum of the magnitudes of h's terms, which partial results are as large as)
        top = torch.where(live[:, t], f[:, t] * top + i[:, t] * v[:, t].abs(), top)
        add = 16 * U * (new.abs() + top + i[:, t] * (v[:, t].abs() + s.abs()))
        e = torch.where(live[:, t], f[:, t] * e + add, e)
        s = torch.where(live[:, t], new, s)
        hs.append(s)
        es.append(e)
    H, EH = torch.stack(hs, 1), torch.stack(es, 1)
    zero = torch.zeros(()).double()
    out = [(torch.where(live, H[:, 1:], zero), torch.where(live, EH[:, 1:], zero)), (s, e)]
    if dh is None and dlast is None:
        return out
    r = dlast.double().cpu() if dlast is not None else torch.zeros(B, D).double()
    dh = dh.double().cpu() if dh is not None else torch.zeros(B, T, D).double()
    er, big = torch.zeros(B, D).double(), r.abs()
    dv, dg, bv, bg = (torch.zeros(B, T, D).double() for _ in range(4))
    for t in range(T - 1, -1, -1):
        on = live[:, t]
        a = r + dh[:, t]
        ea = er + 8 * U * (a.abs() + r.abs())
        d = H[:, t] - v[:, t]
        dv[:, t] = torch.where(on, i[:, t] * a, zero)
        bv[:, t] = torch.where(on, i[:, t] * (ea + 8 * U * a.abs()), zero)
        dg[:, t] = torch.where(on, a * d * i[:, t] * f[:, t], zero)
        # the factor 1 - i is off by an absolute u beside its own rounding
        bg[:, t] = torch.where(on, i[:, t] * (f[:, t] * (ea * d.abs() + a.abs() * EH[:, t] + 16 * U * (a * d).abs())
                                              + 4 * U * (a * d).abs()), zero)
        # r is joined from partial results that are as large as the sum of its terms' magnitudes,
        # whatever r itself cancels to: er obeys the recurrence with |dh| + the magnitude so far
        big = torch.where(on, f[:, t] * (big + dh[:, t].abs()), big)
        er = torch.where(on, f[:, t] * ea + 8 * U * (a.abs() + big), er)
        r = torch.where(on, f[:, t] * a, r)
    return out + [(dv, bv), (dg, bg), (r, er)]


REC_SHAPES = [(1, 1, 1), (3, 1, 40), (2, 2, 7), (1, 3, 8), (5, 7, 5), (2, 8, 64), (3, 9, 65), (2, 16, 33), (4, 50, 32),
              (3, 63, 8), (2, 64, 130), (2, 65, 9), (1, 127, 72), (2, 128, 8), (1, 255, 40), (2, 256, 16), (1, 257, 136),
              (1, 500, 24), (2, 513, 64), (1, 1023, 8), (1, 1030, 264), (1, 2500, 4), (300, 20, 16), (70, 100, 48), (170, 130, 130),
              (1, 1500, 515), (3, 700, 1030), (170, 65, 264), (17000, 11, 16)]


@pytest.mark.parametrize("ragged", [False, True], ids=["", "ragged"])
@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("B,T,D", REC_SHAPES)
def test_gated_recurrence(B, T, D, dtype, ragged):
    v = rnd(B, T, D, dtype=dtype)
    g = rnd(B, T, D, dtype=dtype, mean=2.0, std=2.0)
    h0 = rnd(B, D)
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), device=DEV, dtype=torch.int32)
        lengths[0] = T // 2
        behind = (torch.arange(T, device=DEV) >= lengths.unsqueeze(1)).unsqueeze(2).expand(B, T, D)
        v[behind] = float("nan")     # whatever stands behind the end
        g[behind] = float("inf")
    dh, dlast = rnd(B, T, D, dtype=dtype), rnd(B, D)
    if ragged:
        dh[behind] = float("nan")
    for t in (v, g, h0):
        t.requires_grad_()
    h, last = gated_recurrence(v, g, h0, lengths)
    assert h.dtype == dtype and last.dtype == torch.float32
    grads = torch.autograd.grad((h, last), (v, g, h0), (dh, dlast))
    want = ref_rec(v.detach(), g.detach(), h0.detach(), lengths, dh, dlast)
    for got, (w, b), what in zip((h, last, *grads), want, ("h", "last", "dv", "dg", "dh0")):
        near(got, w, b, what)
    with torch.no_grad():
        h2, last2 = gated_recurrence(v, g, h0, lengths)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    again = torch.autograd.grad(gated_recurrence(v, g, h0, lengths), (v, g, h0), (dh, dlast))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("B,T,D", [(1, 6000, 24), (2, 5000, 1030), (3, 4100, 700)])
def test_recurrence_segments_that_end_anywhere(B, T, D):
    """Long ragged histories, whose time axis is cut: ends in front of, inside and behind a segment,
    on the edge of a tile, and nowhere, with the same bits every time."""
    v, g, h0 = rnd(B, T, D), rnd(B, T, D, mean=1.0), rnd(B, D)
    dh, dlast = rnd(B, T, D), rnd(B, D)
    leaves = [t.requires_grad_() for t in (v, g, h0)]
    for ends in ((0, 1, T), (255, 256, 257), (T - 1, 1000, 1151), (2048, T // 2, 129)):
        lengths = torch.tensor(ends[:B], device=DEV)
        h, last = gated_recurrence(*leaves, lengths)
        got = (h, last, *torch.autograd.grad((h, last), leaves, (dh, dlast)))
        want = ref_rec(v.detach(), g.detach(), h0.detach(), lengths, dh, dlast)
        for a, (w, b), what in zip(got, want, ("h", "last", "dv", "dg", "dh0")):
            near(a, w, b, f"{what} with ends {ends[:B]}")
        for _ in range(3):
            h, last = gated_recurrence(*leaves, lengths)
            again = (h, last, *torch.autograd.grad((h, last), leaves, (dh, dlast)))
            assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("ragged", [False, True], ids=["", "ragged"])
@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("B,T,D", [(3, 9, 1), (5, 33, 16), (4, 64, 17), (2, 65, 32), (7, 128, 3), (3, 129, 8), (300, 200, 12),
                                   (260, 513, 9), (1, 1023, 16), (2, 1024, 31), (1, 1025, 7), (130, 2100, 2), (2, 9000, 10),
                                   (150, 600, 40), (90, 600, 130)])
def test_gated_recurrence_narrow(B, T, D, dtype, ragged):
    """Few channels: one or two tiles of 32 bytes, with and without a cut time axis, and widths just above."""
    test_gated_recurrence(B, T, D, dtype, ragged)


@pytest.mark.parametrize("ragged", [False, True], ids=["", "ragged"])
@pytest.mark.parametrize("dtype,B,T,D", [pytest.param(t, *shape[3:], id="-".join(map(str, (names(t), *shape))))
                                         for t in TYPES for shape in FORMS[t.itemsize]])
def test_gated_recurrence_forms(B, T, D, dtype, ragged):
    """Every form of the kernels in every type (test_sequence.py holds the shapes to their forms)."""
    test_gated_recurrence(B, T, D, dtype, ragged)


def test_narrow_segments_that_end_anywhere():
    """Narrow rows over a cut time axis: the same bits every time, the gradients of the joint input's halves."""
    B, T, D = 2, 7000, 14
    vg, h0 = rnd(B, T, 2 * D).requires_grad_(), rnd(B, D).requires_grad_()
    dh, dlast = rnd(B, T, D), rnd(B, D)
    for ends in ((0, T), (1, 1023), (1024, 1025), (T - 1, 2048), (4096, 6144)):
        lengths = torch.tensor(ends, device=DEV)
        h, last = gated_recurrence(vg, None, h0, lengths)
        dvg, dh0 = torch.autograd.grad((h, last), (vg, h0), (dh, dlast))
        want = ref_rec(vg.detach()[..., :D], vg.detach()[..., D:], h0.detach(), lengths, dh, dlast)
        got = (h, last, dvg[..., :D], dvg[..., D:], dh0)
        for a, (w, b), what in zip(got, want, ("h", "last", "dv", "dg", "dh0")):
            near(a, w, b, f"{what} with ends {ends}")
        for _ in range(3):
            h, last = gated_recurrence(vg, None, h0, lengths)
            dvg, dh0 = torch.autograd.grad((h, last), (vg, h0), (dh, dlast))
            assert all(torch.equal(a, b) for a, b in zip(got, (h, last, dvg[..., :D], dvg[..., D:], dh0)))


@pytest.mark.parametrize("T", [70, 130])
def test_narrow_rows_far_apart(T):
    """Steps 2^23 - 1 elements apart, which is as far as is taken: a wave's offsets come near 2^32 bytes."""
    D, far = 8, 2 ** 23 - 1
    big = torch.empty(1, T, far, device=DEV)
    v, g = big[..., far - D:], big[..., 3:3 + D]
    v.copy_(rnd(1, T, D))
    g.copy_(rnd(1, T, D, mean=1.0))
    dh = rnd(1, T, D)
    apart = [t.detach().requires_grad_() for t in (v, g)]
    dense = [t.detach().contiguous().requires_grad_() for t in (v, g)]
    assert apart[0].stride(1) == far and dense[0].stride(1) == D
    for a, b in zip(*((h, last, *torch.autograd.grad(h, leaves, dh))
                      for leaves in (apart, dense) for h, last in (gated_recurrence(*leaves),))):
        assert torch.equal(a, b)


def test_recurrence_partial_arguments():
    """No state before, one output's gradient only, the joint form, int64 and odd lengths, strides."""
    B, T, D = 3, 70, 24
    vg = rnd(B, T, 2 * D).requires_grad_()
    v, g = vg.detach()[..., :D], vg.detach()[..., D:]
    dh, dlast = rnd(B, T, D), rnd(B, D)
    h, last = gated_recurrence(vg)
    for grads_of, kw in ((((h,), vg, (dh,)), dict(dh=dh)), (((last,), vg, (dlast,)), dict(dlast=dlast))):
        got, = torch.autograd.grad(*grads_of, retain_graph=True)
        want = ref_rec(v, g, None, None, **kw)
        near(got[..., :D], *want[2], "dv")
        near(got[..., D:], *want[3], "dg")
    near(h, *ref_rec(v, g, None, None)[0], "h")
    # strided views, transposed batches, a gradient that is one number expanded
    base = rnd(T, B, 3 * D + 1).requires_grad_()
    tv, tg = base[:, :, 1:D + 1].transpose(0, 1), base[:, :, D + 3:2 * D + 3].transpose(0, 1)
    lengths = torch.tensor([-5, 2 ** 40, 33], device=DEV)
    h, last = gated_recurrence(tv, tg, None, lengths)
    got = torch.autograd.grad(h.sum(), (tv, tg))
    want = ref_rec(tv.detach(), tg.detach(), None, lengths, torch.ones(B, T, D))
    for a, (w, b) in zip((h, last, *got), want):
        near(a, w, b, "strided")
    # no steps, no rows
    z = torch.zeros(B, 0, D, device=DEV, requires_grad=True)
    s = rnd(B, D).requires_grad_()
    h, last = gated_recurrence(z, z, s)
    assert h.shape == (B, 0, D) and torch.equal(last, s)
    assert torch.equal(torch.autograd.grad(last, s, dlast)[0], dlast)
    h, last = gated_recurrence(rnd(0, T, D), rnd(0, T, D))
    assert h.shape == (0, T, D) and last.shape == (0, D)
    # every sequence empty
    none = torch.zeros(B, device=DEV, dtype=torch.int32)
    h, last = gated_recurrence(rnd(B, T, D), rnd(B, T, D), s, none)
    assert not h.any() and torch.equal(last, s)


def test_single_steps_of_time_major_rows():
    """One step of [1, B, D] rows seen as [B, 1, D], 2^23 elements "to the next step", with a gradient
    laid out likewise; through Python and through the C entries with the stride as it is."""
    from recommendsystem_amd import _lib
    B, D = 2 ** 13, 2 ** 10
    v, g, dh = (rnd(1, B, D, dtype=torch.bfloat16).transpose(0, 1) for _ in range(3))
    h0 = rnd(B, D)
    far = v.stride(1)
    assert far == 2 ** 23
    leaves = [t.requires_grad_() for t in (v, g, h0)]
    h, last = gated_recurrence(*leaves)
    got = (h, last, *torch.autograd.grad(h, leaves, dh))
    for a, (w, b), what in zip(got, ref_rec(v.detach(), g.detach(), h0.detach(), None, dh),
                               ("h", "last", "dv", "dg", "dh0")):
        near(a, w, b, what)
    outs = [torch.empty_like(t) for t in got]
    s = torch.cuda.current_stream().cuda_stream
    p = [t.data_ptr() for t in (v, g, h0, *outs)]
    _lib.call("rs_gated_rec_fwd", s, 1, p[0], D, far, p[1], D, far, B, 1, D, None, p[2], p[3], p[4], None, None, 0)
    _lib.call("rs_gated_rec_bwd", s, 1, p[0], D, far, p[1], D, far, B, 1, D, None, p[2], None, dh.data_ptr(), D,
              far, None, p[5], D, far, p[6], D, far, p[7], None, 0)
    for a, b in zip(outs, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,D", [(300, 24), (2000, 8), (5000, 1024)])
def test_recurrence_of_an_empty_batch(T, D):
    """Histories of more than one tile, but none of them: forward and backward of every long form."""
    leaves = [rnd(0, T, D).requires_grad_(), rnd(0, T, D).requires_grad_(), rnd(0, D).requires_grad_()]
    h, last = gated_recurrence(*leaves, torch.zeros(0, device=DEV, dtype=torch.int32))
    assert h.shape == (0, T, D) and last.shape == (0, D)
    for t, grad in zip(leaves, torch.autograd.grad((h, last), leaves, (rnd(0, T, D), rnd(0, D)))):
        assert grad.shape == t.shape


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_recurrence_extreme_gates(dtype):
    """Gates wide open, shut, infinite: i = sigmoid(-g) keeps its own digits where f rounds to 1."""
    B, T, D = 2, 300, 8
    v, h0 = rnd(B, T, D, dtype=dtype), rnd(B, D)
    for gate in (-300.0, -20.0, 0.0, 9.0, 16.5, 60.0, 300.0, float("inf"), float("-inf")):
        g = torch.full((B, T, D), gate, device=DEV).to(dtype).requires_grad_()
        vr = v.clone().requires_grad_()
        h, last = gated_recurrence(vr, g, h0)
        dh = rnd(B, T, D, dtype=dtype)
        got = (h, last, *torch.autograd.grad(h, (vr, g), dh))
        for a, (w, b), what in zip(got, ref_rec(v, g.detach(), h0, None, dh), ("h", "last", "dv", "dg")):
            near(a, w, b + 1e-38, f"{what} at gate {gate}")


def ref_shut(v, g, h0, dh, dlast):
    """(value, bound) pairs as ref_rec's, for gates below 0 with every term of the bound scaled by its own
    factor f or i: f = e^g / (1 + e^g) holds to gate = 12 u of itself (exponential, sum, reciprocal,
    product), for 16-bit rows and 2 |g| u more (the rounded exponent of the hardware's exp2)."""
    B, T, D = v.shape
    gate = U * (12 + (2 * g.double().cpu().abs() if g.dtype != torch.float32 else torch.zeros(())))
    gate = gate.expand(B, T, D)
    v, g, s, dh, r = (t.double().cpu() for t in (v, g, h0, dh, dlast))
    f, i = torch.sigmoid(g), torch.sigmoid(-g)
    e, top = torch.zeros(B, D).double(), s.abs()
    hs, es = [s], [e]
    for t in range(T):
        new = f[:, t] * s + i[:, t] * v[:, t]
        e = f[:, t] * (e + (gate[:, t] + 8 * U) * top) + 8 * U * (i[:, t] * v[:, t].abs() + new.abs())
        top = f[:, t] * top + i[:, t] * v[:, t].abs()
        s = new
        hs.append(s)
        es.append(e)
    H, EH = torch.stack(hs, 1), torch.stack(es, 1)
    out = [(H[:, 1:], EH[:, 1:]), (s, e)]
    er, big = torch.zeros(B, D).double(), r.abs()
    dv, dg, bv, bg = (torch.zeros(B, T, D).double() for _ in range(4))
    for t in range(T - 1, -1, -1):
        a = r + dh[:, t]
        ea = er + 8 * U * (a.abs() + r.abs())
        d = H[:, t] - v[:, t]
        dv[:, t], bv[:, t] = i[:, t] * a, i[:, t] * (ea + 8 * U * a.abs())
        dg[:, t] = a * d * i[:, t] * f[:, t]
        bg[:, t] = i[:, t] * f[:, t] * (ea * d.abs() + a.abs() * (EH[:, t] + U * d.abs())
                                        + (gate[:, t] + 16 * U) * (a * d).abs())
        big = f[:, t] * (big + dh[:, t].abs())
        er = f[:, t] * ea + (gate[:, t] + 8 * U) * (f[:, t] * a.abs() + big)
        r = f[:, t] * a
    return out + [(dv, bv), (dg, bg), (r, er)]


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("B,T,D", [(2, 1, 24), (3, 5, 24), (2, 20, 130), (2, 60, 130), (2, 50, 8), (1, 300, 24), (2, 1100, 8),
                                   (1, 6000, 24), (2, 700, 1000)])
def test_recurrence_of_almost_shut_gates(B, T, D, dtype):
    """f = sigmoid(g) down to e^-30 keeps its own digits: the little of a large state that passes, the
    gradient that reaches it, and the gates' own gradients."""
    v, dh = rnd(B, T, D, dtype=dtype), rnd(B, T, D, dtype=dtype)
    g = (-4 - 26 * torch.rand(B, T, D, device=DEV)).to(dtype)
    h0, dlast = 1e5 * rnd(B, D), 1e5 * rnd(B, D)
    leaves = [t.clone().requires_grad_() for t in (v, g, h0)]
    h, last = gated_recurrence(*leaves)
    got = (h, last, *torch.autograd.grad((h, last), leaves, (dh, dlast)))
    for a, (w, b), what in zip(got, ref_shut(v, g, h0, dh, dlast), ("h", "last", "dv", "dg", "dh0")):
        if dtype is torch.float16 and a.dtype == dtype:
            # dlast times i passes fp16's largest number, 65504: from 65520 on the nearest is infinity
            over = (w.abs() - b > 65520).to(DEV)
            assert torch.equal(a[over], w.to(dtype).to(DEV)[over]) and bool(a[over].isinf().all())
            a, w, b = (torch.where(over.to(t.device) | ((w.abs() + b).to(t.device) > 65504), 0, t) for t in (a, w, b))
        near(a, w, b + 1e-36, what)
    h, new = gated_recurrence_step(v[:, 0], g[:, 0], h0)
    one = ref_shut(v[:, :1], g[:, :1], h0, dh[:, :1], dlast)
    near(h, one[0][0][:, 0], one[0][1][:, 0], "step")
    near(new, *one[1], "step's state")


def test_recurrence_large_state_is_forgotten():
    """A state of 10^6 in front of values around 1, half of it forgotten a step: its rounding is
    forgotten with it, in the states and (from the other end) in the gradients."""
    B, T, D = 1, 700, 16
    v, g, dh = rnd(B, T, D), rnd(B, T, D, std=0.1).requires_grad_(), rnd(B, T, D)
    h0, dlast = 1e6 * rnd(B, D), 1e6 * rnd(B, D)
    vr = v.clone().requires_grad_()
    h, last = gated_recurrence(vr, g, h0)
    got = (h, last, *torch.autograd.grad((h, last), (vr, g), (dh, dlast)))
    for a, (w, b) in zip(got, ref_rec(v, g.detach(), h0, None, dh, dlast)):
        near(a, w, b, "large state")


@pytest.mark.parametrize("dtype", TYPES, ids=names)
@pytest.mark.parametrize("T,D", [(5, 24), (20, 130), (50, 130), (50, 8), (200, 24), (300, 24), (1100, 8), (3000, 24)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_behind_the_end_have_no_gradient(bad, T, D, dtype):
    """An overflowed gradient of the last state reaches the steps of its channel, and none behind the end."""
    v, g = rnd(3, T, D, dtype=dtype).requires_grad_(), rnd(3, T, D, dtype=dtype).requires_grad_()
    lengths = torch.tensor([T - 2, 0, T // 2], device=DEV)
    h, last = gated_recurrence(v, g, None, lengths)
    dlast = rnd(3, D)
    dlast[:, 1] = bad
    for grad in torch.autograd.grad((h, last), (v, g), (rnd(3, T, D, dtype=dtype), dlast)):
        for b, n in enumerate(lengths.tolist()):
            assert not grad[b, n:].any() and not grad[b, n:].isnan().any()
            assert n == 0 or not grad[b, n - 1, 1].isfinite()


def test_recurrence_nan_stays_in_its_channel():
    v, g = rnd(2, 100, 20), rnd(2, 100, 20)
    v[0, 50, 3] = float("nan")
    h, last = gated_recurrence(v, g)
    want = torch.zeros(2, 100, 20, dtype=torch.bool)
    want[0, 50:, 3] = True
    assert torch.equal(h.isnan().cpu(), want)


def test_recurrence_differences():
    """Against central differences: the step's own error is h^2/6 of a third derivative (the state
    is a product of at most 40 sigmoids, its third derivative along a unit direction of order 1)
    and the rounding over h: 1e-3 of the gradient's norm covers both."""
    v, g, h0 = rnd(2, 40, 6), rnd(2, 40, 6), rnd(2, 6)
    dh, dl = rnd(2, 40, 6), rnd(2, 6)
    leaves = [t.clone().requires_grad_() for t in (v, g, h0)]
    grads = torch.autograd.grad(gated_recurrence(*leaves), leaves, (dh, dl))

    def loss(*a):
        h, last = gated_recurrence(*a)
        return float((h.double() * dh.double()).sum() + (last.double() * dl.double()).sum())
    for k, t in enumerate((v, g, h0)):
        d = rnd(*t.shape)
        d /= d.norm()
        h = 2.0 ** -5
        args = lambda s: [p + s * d if i == k else p for i, p in enumerate((v, g, h0))]  # noqa: E731
        diff = (loss(*args(h)) - loss(*args(-h))) / (2 * h)
        assert abs(diff - float((grads[k] * d).double().sum())) <= 1e-3 * float(grads[k].norm())


@pytest.mark.parametrize("dtype", TYPES, ids=names)
def test_step_matches_the_recurrence(dtype):
    B, T, D = 5, 11, 37
    v, g, h0 = rnd(B, T, D, dtype=dtype), rnd(B, T, D, dtype=dtype, mean=1.0), rnd(B, D)
    want = ref_rec(v, g, h0, None)
    state = h0.clone()
    for t in range(T):
        h, new = gated_recurrence_step(v[:, t], g[:, t], state, state)  # in place
        assert new.data_ptr() == state.data_ptr() and h.dtype == dtype
        near(h, want[0][0][:, t], want[0][1][:, t], f"step {t}")
    near(state, *want[1], "state")
    vg = torch.cat([v[:, 0], g[:, 0]], 1)
    h, new = gated_recurrence_step(vg)
    first = ref_rec(v[:, :1], g[:, :1], None, None)
    near(h, first[0][0][:, 0], first[0][1][:, 0], "joint, no state")
    near(new, *first[1], "joint, no state")
    h, new = gated_recurrence_step(v[:0, 0], g[:0, 0])
    assert h.shape == (0, D)


def test_step_output_that_overlaps_is_refused():
    m, v = torch.zeros(96, device=DEV), rnd(5, 8)
    state, out = m[:40].view(5, 8), m[8:48].view(5, 8)
    with pytest.raises(ValueError, match="overlaps the state"):
        gated_recurrence_step(v, v, state, out)
    with pytest.raises(ValueError, match="overlaps the values"):
        gated_recurrence_step(out, v, None, out.view(5, 8))
    h, new = gated_recurrence_step(v, v, state, state.view(5, 8))     # another tensor of the same memory
    assert new.data_ptr() == state.data_ptr() and torch.equal(state, h)
    gated_recurrence_step(v, v, state, m[40:80].view(5, 8))


# ============================================================================================
# streams, graphs, large tensors
# ============================================================================================
def test_other_stream():
    x, g = rnd(200, 64).view(4, 50, 64), rnd(4, 50, 64)
    gamma, beta = rnd(64), rnd(64)
    want = gated_recurrence(layer_norm(x, gamma, beta), g)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gated_recurrence(layer_norm(x, gamma, beta), g)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_captured_training_step():
    """Forward and backward of all three in one graph, replayed on new inputs with eager work of
    the same kind between the replays; a second graph of the same calls beside it."""
    B, T, D = 2, 300, 40

    def step(x, gate, gamma, beta, dh):
        y = layer_norm(x, gamma, beta, 1e-5, True)
        h, last = gated_recurrence(y, gate)
        grads = torch.autograd.grad((h, last), (x, gate, gamma, beta), (dh, torch.ones_like(last)))
        return (h, last, *grads, *pack8(h))
    ins = [rnd(B, T, D).requires_grad_(), rnd(B, T, D).requires_grad_(), rnd(D).requires_grad_(),
           rnd(D).requires_grad_(), rnd(B, T, D)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*ins)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step(*ins)
        graphs.append((gr, outs))
    for k in range(4):
        with torch.no_grad():
            for t in ins:
                t.copy_(rnd(*t.shape))
        for gr, _ in graphs:
            gr.replay()
        fresh = [t.detach().clone().requires_grad_(t.requires_grad) for t in ins]
        want = step(*fresh)
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), f"replay {k}"


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows against the same rows by themselves."""
    D = 1024
    R = 2 ** 21 + 5
    x = torch.empty(R, D, device=DEV, dtype=torch.bfloat16).normal_()
    gamma, beta = rnd(D), rnd(D)
    xr = x.requires_grad_()
    y = layer_norm(xr, gamma, beta, 1e-5, True)
    dx, = torch.autograd.grad(y, xr, x.detach())
    tail = x.detach()[-70:].clone().requires_grad_()
    yt = layer_norm(tail, gamma, beta, 1e-5, True)
    assert torch.equal(y[-70:], yt)
    assert torch.equal(dx[-70:], torch.autograd.grad(yt, tail, tail.detach())[0])
    del y, dx, xr
    x = x.detach()
    codes, scales = pack8(x)
    ct, st = pack8(x[-9:].clone())
    assert torch.equal(codes[-9:], ct) and torch.equal(scales[-9:], st)
    assert torch.equal(unpack8(codes, scales, torch.bfloat16)[-9:], unpack8(ct, st, torch.bfloat16))
    del codes, scales
    # one history of 2^21 events; gates around 0 forget within some tens of steps
    # (values and gates are two leaves of one memory: summed, their gradients would be rounded to
    # the type once more, and cancel)
    v, g = x.view(1, R, D).requires_grad_(), x.view(1, R, D).detach().requires_grad_()
    h, last = gated_recurrence(v, g)
    dv, dg = torch.autograd.grad((h, last), (v, g), (v.detach(), torch.ones_like(last)))
    tv, tg = (t.detach()[:, -400:].clone().requires_grad_() for t in (v, g))
    th, tlast = gated_recurrence(tv, tg)
    tdv, tdg = torch.autograd.grad((th, tlast), (tv, tg), (tv.detach(), torch.ones_like(tlast)))
    # fp32 values that differ in their last digits round to neighbours: one step of the type
    for a, b in ((h[:, -200:], th[:, -200:]), (dv[:, -200:], tdv[:, -200:]), (dg[:, -200:], tdg[:, -200:])):
        assert bool(((a.float() - b.float()).abs() <= 2 * 2.0 ** -8 * b.float().abs() + 1e-5).all())
    near(last, tlast.double().cpu(), 64 * U * (1 + tlast.double().cpu().abs()), "last")


# ============================================================================================
# together: the encoder, Dense with an 8-bit input, the custom operators
# ============================================================================================
def test_second_derivatives_are_refused():
    """create_graph gives the same first derivatives; asking for a second raises."""
    x, g = rnd(2, 9, 12).requires_grad_(), rnd(2, 9, 12).requires_grad_()
    gamma, beta = rnd(12).requires_grad_(), rnd(12).requires_grad_()
    for run in (lambda: layer_norm(x, gamma, beta), lambda: layer_norm(x, gamma, beta, 1e-5, True),
                lambda: gated_recurrence(x, g)[0]):
        want, = torch.autograd.grad(run().square().sum(), x)
        got, = torch.autograd.grad(run().square().sum(), x, create_graph=True)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            got.sum().backward()


def test_inference_mode_and_two_streams():
    """Under inference mode, and two calls in flight at once."""
    x, g = rnd(3, 5000, 64), rnd(3, 5000, 64)
    gamma, beta = rnd(64), rnd(64)
    want = gated_recurrence(layer_norm(x, gamma, beta), g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    with torch.inference_mode():
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append([gated_recurrence(layer_norm(x, gamma, beta), g) for _ in range(4)])
        torch.cuda.synchronize()
    for run in outs:
        for h, last in run:
            assert torch.equal(h, want[0]) and torch.equal(last, want[1])


def test_dense_save_8bit():
    a, b = Dense(20, "relu", seed=3), Dense(20, "relu", seed=3, save_8bit=True)
    x = rnd(65, 300)
    dy = rnd(65, 20)
    xa, xb = x.clone().requires_grad_(), x.clone().requires_grad_()
    ya, yb = a(xa), b(xb)
    assert torch.equal(ya, yb)
    ya.backward(dy)
    yb.backward(dy)
    assert torch.equal(xa.grad, xb.grad) and torch.equal(a.bias.grad, b.bias.grad)
    c = Dense(20, "relu", seed=3)   # the same kernel gradient from the kept values themselves
    c.build((300,), device=x.device)
    kept = unpack8(*pack8(x))
    dz = dy.double() * (ya > 0)
    want = (kept.double().t() @ dz).cpu()
    bound = 64 * U * (kept.double().abs().t() @ dz.abs()).cpu()
    near(b.kernel.grad, want, bound, "dW")
    err = (b.kernel.grad - a.kernel.grad).abs()   # half a step of every kept value
    step = pack8(x)[1].repeat_interleave(128, 1)[:, :300] / 2
    assert bool((err <= step.t() @ dz.abs().float() * 1.001 + 1e-4).all())


def test_dense_save_8bit_packs_only_for_a_kernel_gradient(monkeypatch):
    """A frozen layer passes its input's gradient on without its input, and its gradient buffers are left
    alone; a forward without any gradient, and a group of layers in inference, keep nothing either."""
    from recommendsystem_amd import layers
    packed = []
    monkeypatch.setattr(layers, "pack8", lambda x: (packed.append(1), pack8(x))[1])
    a, b = Dense(20, "relu", seed=3), Dense(20, "relu", seed=3, save_8bit=True)
    x, dy = rnd(65, 300), rnd(65, 20)
    xa, xb = x.clone().requires_grad_(), x.clone().requires_grad_()
    a(xa).backward(dy)
    y = b(x)
    assert len(packed) == 1                   # (its parameters want gradients)
    for p in b.parameters():
        p.requires_grad_(False)
    grads = [t.grad.fill_(7.0) for t in (b.kernel, b.bias)]
    assert torch.equal(b(xb), y)
    b(xb).backward(dy)
    dz = dy.double() * (y > 0)
    near(xb.grad, (dz @ a.kernel.detach().double().t()).cpu(), 64 * U * (dz.abs() @ a.kernel.detach().double().abs().t()).cpu(), "dx")
    near(xa.grad, (dz @ a.kernel.detach().double().t()).cpu(), 64 * U * (dz.abs() @ a.kernel.detach().double().abs().t()).cpu(), "dx")
    assert all(bool((t == 7.0).all()) for t in grads) and not b(x).requires_grad
    sink = layers.GradSink()                  # the producer's gradient is added onto
    sink.buf = dx = rnd(65, 300)
    want = dx.double().cpu() + xb.grad.double().cpu()
    xs = x.clone().requires_grad_()
    b(xs, sink).backward(dy)
    near(xs.grad, want, 4 * U * (want.abs() + xb.grad.double().cpu().abs()), "dx onto a sink's")
    c = Dense(20, "relu", seed=4, save_8bit=True)
    with torch.no_grad():
        for got, layer in zip(layers.grouped_dense([b, c], [x, x]), (b, c)):
            near(got, layer(x).double().cpu(), 64 * U * (x.double().abs() @ layer.kernel.double().abs()).cpu(), "grouped")
    assert len(packed) == 1


def plain_encoder(enc, x, lengths, states, dtype=torch.float64):
    """SequenceEncoder from elementary operations in float64, for autograd on the CPU."""
    p = {k: t.detach().cpu().to(dtype).requires_grad_() for k, t in enc.named_parameters()}

    def norm(z, name):
        m = z.mean(-1, keepdim=True)
        return (z - m) / torch.sqrt((z - m).pow(2).mean(-1, keepdim=True) + 1e-5) * p[name + ".gamma"] + p[name + ".beta"]
    B, T, _ = x.shape
    live = torch.arange(T).unsqueeze(0) < lengths.unsqueeze(1)
    x = torch.where(live.unsqueeze(2), x, torch.zeros((), dtype=dtype))
    last = []
    for k in range(enc.depth):
        vg = norm(x, f"norms.{k}") @ p[f"recurrences.{k}.projection.kernel"] + p[f"recurrences.{k}.projection.bias"]
        v, f = vg[..., :enc.units], torch.sigmoid(vg[..., enc.units:])
        s, hs = states[k], []
        for t in range(T):
            s = torch.where(live[:, t:t + 1], f[:, t] * s + (1 - f[:, t]) * v[:, t], s)
            hs.append(torch.where(live[:, t:t + 1], s, torch.zeros((), dtype=dtype)))
        last.append(s)
        x = x + torch.stack(hs, 1) @ p[f"outputs.{k}.kernel"] + p[f"outputs.{k}.bias"]
    y = norm(x, "final")
    return torch.where(live.unsqueeze(2), y, torch.zeros((), dtype=dtype)), torch.stack(last), p


@pytest.mark.parametrize("save_8bit", [False, True], ids=["", "8bit"])
def test_encoder(save_8bit):
    """Values to 1e-4 (fp32 through 2 blocks of sums over at most 48 terms), gradients to 1e-3 of
    their largest; with 8-bit inputs every kept value is off by at most 1/254 of its block's largest,
    which leaves the gradients within 5 percent of their norm."""
    B, T, E, N = 4, 70, 24, 40
    enc = SequenceEncoder(N, depth=2, save_8bit=save_8bit)
    x = rnd(B, T, E)
    lengths = torch.tensor([70, 0, 33, 64], device=DEV)
    x[3, 64:] = float("nan")
    states = rnd(2, B, N)
    xr = x.clone().requires_grad_()
    y, last = enc(xr, lengths, states)
    dy, dl = rnd(B, T, E), rnd(2, B, N)
    (y * dy).sum().add((last * dl).sum()).backward()
    xc = x.double().cpu().requires_grad_()
    yc, lc, p = plain_encoder(enc, xc, lengths.cpu(), states.double().cpu())
    (yc * dy.double().cpu()).sum().add((lc * dl.double().cpu()).sum()).backward()
    assert float((y.detach().double().cpu() - yc.detach()).abs().max()) <= 1e-4
    assert float((last.detach().double().cpu() - lc.detach()).abs().max()) <= 1e-4
    assert not y[1].any() and not xr.grad[1].any() and not xr.grad[3, 64:].any()
    for name, got, want in [("x", xr.grad, xc.grad)] + [(k, t.grad, p[k].grad) for k, t in enc.named_parameters()]:
        got = got.double().cpu()
        assert bool(got.isfinite().all()), name
        if save_8bit:
            assert float((got - want).norm()) <= 0.05 * float(want.norm()), name
        else:
            assert float((got - want).abs().max()) <= 1e-3 * float(want.abs().max()), name


def test_encoder_steps_continue_a_history():
    enc = SequenceEncoder(40, depth=2)
    x = rnd(3, 30, 24)
    with torch.no_grad():
        whole, end = enc(x)
        _, states = enc(x[:, :25], states=None)
        for t in range(25, 30):
            y, states = enc.step(x[:, t], states)
            assert float((y - whole[:, t]).abs().max()) <= 1e-4
        assert float((states - end).abs().max()) <= 1e-4


def test_gated_recurrence_layer_trains_its_projection():
    layer = GatedRecurrence(12, save_8bit=True)
    x = rnd(3, 20, 10).requires_grad_()
    h, last = layer(x, torch.tensor([20, 1, 7], device=DEV, dtype=torch.int32))
    assert h.shape == (3, 20, 12) and float(layer.projection.bias.detach()[12:].min()) == 2.0
    (h.sum() + last.sum()).backward()
    assert bool(layer.projection.kernel.grad.isfinite().all()) and layer.projection.kernel.grad.any()
    assert not x.grad[1, 1:].any()


def test_custom_operators():
    from recommendsystem_amd import ops
    x = rnd(3, 9, 30).requires_grad_()
    gamma, beta = rnd(30).requires_grad_(), rnd(30).requires_grad_()
    torch.library.opcheck(torch.ops.ctr.layer_norm.default, (x, gamma, beta, 1e-5))
    h0 = rnd(3, 30).requires_grad_()
    lengths = torch.tensor([9, 0, 4], device=DEV, dtype=torch.int32)
    g = rnd(3, 9, 30).requires_grad_()
    torch.library.opcheck(torch.ops.ctr.gated_recurrence.default, (x, g, h0, lengths))
    torch.library.opcheck(torch.ops.ctr.gated_recurrence.default, (x, None, None, None))
    torch.library.opcheck(torch.ops.ctr.pack8.default, (x.detach(),))
    torch.library.opcheck(torch.ops.ctr.unpack8.default, (*pack8(x), torch.float32))

    def run():
        h, last = gated_recurrence(layer_norm(x, gamma, beta), g, h0, lengths)
        return (h, last, *torch.autograd.grad(h.sum() + last.sum(), (x, gamma, beta, g, h0)))
    want = run()
    ops.use_custom_ops(True)
    try:
        got = run()
    finally:
        ops.use_custom_ops(False)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_custom_operators_without_gradients():
    """Inference through the operators: the same bits as without them; the step in place as well."""
    from recommendsystem_amd import ops
    x, g = rnd(3, 300, 40), rnd(3, 300, 40)
    gamma, beta, h0 = rnd(40), rnd(40), rnd(3, 40)
    lengths = torch.tensor([300, 0, 77], device=DEV)
    enc = SequenceEncoder(16, depth=2, save_8bit=True)
    for op, args in ((torch.ops.ctr.gated_recurrence_step, (x[:, 0], g[:, 0], h0)),
                     (torch.ops.ctr.gated_recurrence_step, (x[:, 0], None, None))):
        torch.library.opcheck(op.default, args)

    def run():
        state = h0.clone()
        h, new = gated_recurrence_step(x[:, 0], g[:, 0], state, state)
        assert new is state
        with torch.no_grad():
            y, states = enc(x, lengths)
            return (layer_norm(x, gamma, beta), *gated_recurrence(x, g, h0, lengths), h, new, y, states,
                    *enc.step(x[:, 1], states))
    want = run()
    ops.use_custom_ops(True)
    try:
        got = run()
    finally:
        ops.use_custom_ops(False)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
