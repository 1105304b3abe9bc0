"""CPU: the sequence operators' refusals (all of them raise before anything is launched), size
queries and meta shapes."""
import pytest
import torch

from recommendsystem_amd import _lib, packing, sequence
from recommendsystem_amd import ops  # noqa: F401
from recommendsystem_amd.layers import Dense
from _rec_forms import FORMS, STEPS

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
E = torch.empty


@pytest.mark.parametrize("call, error, text", [
    (lambda: sequence.layer_norm(E(3, 4, dtype=F64), E(4), E(4)), TypeError, "float32, bfloat16"),
    (lambda: sequence.layer_norm(E(()), E(4), E(4)), ValueError, "last dimension"),
    (lambda: sequence.layer_norm(E(3, 0), E(0), E(0)), ValueError, "last dimension"),
    (lambda: sequence.layer_norm(E(1, 32769), E(32769), E(32769)), ValueError, "1 to 32768"),
    (lambda: sequence.layer_norm(E(3, 4), E(5), E(4)), ValueError, "gamma"),
    (lambda: sequence.layer_norm(E(3, 4), E(4), E(1, 4)), ValueError, "beta"),
    (lambda: sequence.layer_norm(E(3, 4, dtype=BF16), E(4, dtype=BF16), E(4)), TypeError, "gamma"),
    (lambda: sequence.layer_norm(E(3, 4), E(4), E(4), 0.0), ValueError, "epsilon"),
    (lambda: sequence.layer_norm(E(3, 4), E(4), E(4), float("nan")), ValueError, "epsilon"),
    (lambda: sequence.gated_recurrence(E(2, 3), E(2, 3)), ValueError, "rank-3"),
    (lambda: sequence.gated_recurrence(E(2, 3, 4), E(2, 3, 5)), ValueError, "differ in shape"),
    (lambda: sequence.gated_recurrence(E(2, 3, 4), E(2, 3, 4, dtype=F16)), TypeError, "differ in type"),
    (lambda: sequence.gated_recurrence(E(2, 3, 4, dtype=torch.int32), E(2, 3, 4)), TypeError, "values"),
    (lambda: sequence.gated_recurrence(E(2, 3, 0), E(2, 3, 0)), ValueError, "last dimension"),
    (lambda: sequence.gated_recurrence(E(2, 3, 5)), ValueError, "even"),
    (lambda: sequence.gated_recurrence(E(2, 3, 0)), ValueError, "even"),
    (lambda: sequence.gated_recurrence(E(2, 3, 4), E(2, 3, 4), E(2, 5)), ValueError, "h0"),
    (lambda: sequence.gated_recurrence(E(2, 3, 4), E(2, 3, 4), E(2, 4, dtype=BF16)), TypeError, "h0"),
    (lambda: sequence.gated_recurrence_step(E(2, 3, 4), E(2, 3, 4)), ValueError, "rank-2"),
    (lambda: sequence.gated_recurrence_step(E(2, 4), E(2, 4), E(3, 4)), ValueError, "state"),
    (lambda: sequence.gated_recurrence_step(E(2, 4), E(2, 4), None, E(4, 2).t()), ValueError, "contiguous"),
    (lambda: sequence.gated_recurrence_step(E(2, 4, requires_grad=True), E(2, 4)), RuntimeError, "no backward"),
    (lambda: sequence.pack8(E(3, 4, dtype=torch.int32)), TypeError, "float32"),
    (lambda: sequence.pack8(E(3, 0)), ValueError, "last dimension"),
    (lambda: sequence.unpack8(E(3, 4), E(3, 1)), TypeError, "int8"),
    (lambda: sequence.unpack8(E(3, 4, dtype=torch.int8), E(3, 2)), ValueError, "do not fit"),
    (lambda: sequence.unpack8(E(3, 4, dtype=torch.int8), E(3, 1), F64), TypeError, "dtype"),
    (lambda: sequence.GatedRecurrence(0), ValueError, "unit"),
    (lambda: sequence.GatedRecurrence(4)(E(2, 3)), ValueError, "rank of input"),
    (lambda: sequence.SequenceEncoder(4, depth=0), ValueError, "depth"),
    (lambda: sequence.SequenceEncoder(4)(E(2, 3)), ValueError, "rank of input"),
    (lambda: sequence.SequenceEncoder(4)(E(2, 3, 5), None, E(1, 2, 5)), ValueError, "states"),
])
def test_refusals(call, error, text):
    with pytest.raises(error, match=text):
        call()


@pytest.mark.parametrize("call", [
    lambda: sequence.layer_norm(E(3, 4), E(4), E(4)),
    lambda: sequence.gated_recurrence(E(2, 3, 4), E(2, 3, 4)),
    lambda: sequence.gated_recurrence_step(E(2, 4), E(2, 4)),
    lambda: sequence.pack8(E(3, 4)),
    lambda: sequence.unpack8(E(3, 4, dtype=torch.int8), E(3, 1)),
])
def test_no_cpu_fallback(call):
    with pytest.raises(_lib.RecsysKernelError, match="ROCm device"):
        call()


NORM_BWD = dict(dy=(E, (3, 4)), x=(E, (3, 4)), gamma=(E, (4,)), stats=(E, (2, 3)))
# (the first width of this length that keeps states)
REC_BWD = dict(dh=(E, (2, 300, 40)), dlast=(E, (2, 40)), v=(E, (2, 300, 40)), g=(E, (2, 300, 40)), h0=(E, (2, 40)),
               lengths=None, states=(E, (_lib.load().rs_gated_rec_states_floats(0, 2, 300, 40),)))


@pytest.mark.parametrize("op, args, name, shape, dtype, error", [
    ("layer_norm_bwd", NORM_BWD, "dy", (3, 4), BF16, TypeError),
    ("layer_norm_bwd", NORM_BWD, "dy", (2, 4), F32, ValueError),
    ("layer_norm_bwd", NORM_BWD, "x", (3, 4), F16, TypeError),
    ("layer_norm_bwd", NORM_BWD, "x", (3, 4), F64, TypeError),
    ("layer_norm_bwd", NORM_BWD, "gamma", (3,), F32, ValueError),
    ("layer_norm_bwd", NORM_BWD, "gamma", (4,), BF16, TypeError),
    ("layer_norm_bwd", NORM_BWD, "stats", (2, 2), F32, ValueError),
    ("layer_norm_bwd", NORM_BWD, "stats", (2, 3), F16, TypeError),
    ("gated_recurrence_bwd", REC_BWD, "dh", (2, 300, 40), F16, TypeError),
    ("gated_recurrence_bwd", REC_BWD, "dh", (2, 299, 40), F32, ValueError),
    ("gated_recurrence_bwd", REC_BWD, "dlast", (2, 40), BF16, TypeError),
    ("gated_recurrence_bwd", REC_BWD, "dlast", (1, 40), F32, ValueError),
    ("gated_recurrence_bwd", REC_BWD, "g", (2, 300, 40), BF16, TypeError),
    ("gated_recurrence_bwd", REC_BWD, "g", (2, 300, 39), F32, ValueError),
    ("gated_recurrence_bwd", REC_BWD, "h0", (2, 39), F32, ValueError),
    ("gated_recurrence_bwd", REC_BWD, "h0", (2, 40), F16, TypeError),
    ("gated_recurrence_bwd", REC_BWD, "lengths", (3,), torch.int32, ValueError),
    ("gated_recurrence_bwd", REC_BWD, "lengths", (2,), F32, TypeError),
    ("gated_recurrence_bwd", REC_BWD, "states", (79,), F32, ValueError),
    ("gated_recurrence_bwd", REC_BWD, "states", (0,), F32, ValueError),
    ("gated_recurrence_bwd", REC_BWD, "states", (160,), BF16, TypeError),
])
def test_backward_operators_refuse_what_does_not_fit(op, args, name, shape, dtype, error):
    """They read every argument through its raw pointer, with sizes taken from one of them."""
    made = {k: a and a[0](*a[1]) for k, a in args.items()}
    made[name] = E(shape, dtype=dtype)
    with pytest.raises(error):
        getattr(torch.ops.ctr, op)(*made.values())


@pytest.mark.parametrize("op, args", [("layer_norm_bwd", NORM_BWD), ("gated_recurrence_bwd", REC_BWD)])
def test_backward_operators_take_what_fits(op, args):
    with pytest.raises(_lib.RecsysKernelError, match="ROCm device"):  # the next check after the sizes
        getattr(torch.ops.ctr, op)(*(a and a[0](*a[1]) for a in args.values()))


def dual(*shape):
    return torch.autograd.forward_ad.make_dual(torch.ones(*shape), torch.ones(*shape))


@pytest.mark.parametrize("call", [
    lambda: sequence.layer_norm(dual(3, 4), E(4), E(4)),
    lambda: sequence.layer_norm(E(3, 4), dual(4), E(4), save_8bit=True),
    lambda: sequence.layer_norm(E(3, 4), E(4), dual(4)),
    lambda: sequence.gated_recurrence(dual(2, 3, 4), E(2, 3, 4)),
    lambda: sequence.gated_recurrence(E(2, 3, 4), dual(2, 3, 4)),
    lambda: sequence.gated_recurrence(dual(2, 3, 4)),
    lambda: sequence.gated_recurrence(E(2, 3, 4), E(2, 3, 4), dual(2, 4)),
    lambda: sequence.gated_recurrence_step(dual(2, 4), E(2, 4)),
    lambda: sequence.gated_recurrence_step(E(2, 4), E(2, 4), dual(2, 4)),
    lambda: torch.ops.ctr.layer_norm(dual(3, 4), E(4), E(4), 1e-5),
    lambda: torch.ops.ctr.gated_recurrence(dual(2, 3, 4), None, None, None),
])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(call, grad):
    """Not dropped: without a jvp the output would come back with no tangent and no word."""
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="jvp"):
            call()


def test_tangents_of_others_do_not_matter():
    with pytest.raises(NotImplementedError, match="jvp"):
        torch.func.jvp(lambda x: sequence.layer_norm(x, E(4), E(4)), (E(3, 4),), (E(3, 4),))
    with torch.autograd.forward_ad.dual_level():
        dual(3, 4)
        with pytest.raises(_lib.RecsysKernelError, match="ROCm device"):
            sequence.layer_norm(E(3, 4), E(4), E(4))


def test_lengths_checks():
    for bad, err in ((E(3), TypeError), (E(4, dtype=torch.int32), ValueError),
                     (E(3, 1, dtype=torch.int32), ValueError)):
        with pytest.raises(err, match="lengths"):
            sequence._check_lengths(bad, 3, 5)
    got = sequence._check_lengths(torch.tensor([2 ** 32 + 1, -7, 3]), 3, 5)
    assert got.dtype == torch.int32 and got.tolist() == [5, 0, 3]


def test_strides_of_a_single_step():
    """A [B, 1, D] view of time-major [1, B, D] rows says B D elements to the next step, and counts as
    contiguous: there is no next step, so nothing has to be copied and nothing is refused."""
    far = E(1, 8192, 1024, device="meta").transpose(0, 1)
    assert far.stride(1) >= sequence.MAX_STEP_STRIDE
    t, sb, st = sequence._strided(far)
    assert t is far and sb == 1024 and st < sequence.MAX_STEP_STRIDE
    two = E(2, 8192, 1024, device="meta").transpose(0, 1)      # with a next step it is copied
    assert sequence._strided(two)[1:] == (2048, 1024)
    # the C entries: a step stride that is too long is refused where there are two steps
    lib, p, far = _lib.load(), torch.zeros(64).data_ptr(), 1 << 23
    UNS = _lib.RS_ERR_UNSUPPORTED
    assert lib.rs_gated_rec_fwd(None, 0, p, 4, far, p, 4, 4, 1, 2, 4, None, None, p, p, None, None, 0) == UNS
    assert lib.rs_gated_rec_bwd(None, 0, p, 4, 4, p, 4, 4, 1, 2, 4, None, None, None, p, 4, far, p, p, 4, 4, p,
                                4, 4, p, None, 0) == UNS


def test_entry_points_reject():
    """The C entry points refuse what they cannot run before they launch (null or short buffers)."""
    lib = _lib.load()
    some = torch.zeros(64)
    p = some.data_ptr()
    ARG, UNS = _lib.RS_ERR_ARG, _lib.RS_ERR_UNSUPPORTED
    assert lib.rs_pack8(None, 3, p, 4, 1, 4, p, p) == ARG           # type
    assert lib.rs_pack8(None, 0, None, 4, 1, 4, p, p) == ARG
    assert lib.rs_pack8(None, 0, p, 4, 1, 0, p, p) == ARG
    assert lib.rs_pack8(None, 0, p, 4, 1, (1 << 30) + 1, p, p) == ARG
    assert lib.rs_pack8(None, 0, None, 4, 0, 4, None, None) == 0    # no rows
    assert lib.rs_unpack8(None, 0, p, p, 1, 4, p, 3) == ARG         # ld_y < D
    assert lib.rs_layernorm_fwd(None, 0, p, 4, 1, 32769, p, p, 1e-5, p, 32769, None, None, None, None) == UNS
    assert lib.rs_layernorm_fwd(None, 0, p, 4, 1, 4, p, p, 0.0, p, 4, None, None, None, None) == ARG
    assert lib.rs_layernorm_fwd(None, 0, p, 4, 1, 4, p, p, 1e-5, p, 4, p, None, None, None) == ARG
    assert lib.rs_layernorm_fwd(None, 0, p, 4, 1, 4, p, p, 1e-5, p, 4, None, None, p, None) == ARG
    need = lib.rs_layernorm_bwd_workspace_floats(1000, 4)
    assert lib.rs_layernorm_bwd(None, 0, p, 4, p, 4, None, None, 1000, 4, p, p, p, p, 4, p, p, 0, p, need - 1) == ARG
    assert lib.rs_layernorm_bwd(None, 0, p, 4, p, 4, p, p, 1, 4, p, p, p, p, 4, p, p, 0, p, 64) == ARG  # both
    assert lib.rs_gated_rec_fwd(None, 0, p, 4, 4, p, 4, 4, 1, -1, 4, None, None, p, p, None, None, 0) == ARG
    assert lib.rs_gated_rec_fwd(None, 0, p, 4, 4, p, 4, 4, 1, 1, 4, None, None, p, None, None, None, 0) == ARG
    assert lib.rs_gated_rec_fwd(None, 0, p, 4, 4, p, 4, 4, 0, 9, 4, None, None, None, None, None, None, 0) == 0
    assert lib.rs_gated_rec_bwd(None, 0, p, 4, 4, p, 4, 4, 1, 999, 4, None, None, None, p, 4, 4, p, p, 4, 4, p,
                                4, 4, p, None, 0) == ARG             # no states
    assert lib.rs_gated_rec_step(None, 0, p, 4, p, 4, 1, 4, p, p, None) == ARG
    # a workspace that the shape needs and that is missing
    B, T, D = 1, 1 << 20, 8
    if lib.rs_gated_rec_workspace_floats(0, B, T, D):
        assert lib.rs_gated_rec_fwd(None, 0, p, 8, 8, p, 8, 8, B, T, D, None, None, p, p, None, None, 0) == ARG


def test_size_queries():
    lib = _lib.load()
    for B, T, D in ((1, 1, 1), (3, 50, 32), (1, 1 << 20, 1000), (70000, 3, 5), (8, 4096, 2048)):
        for code in (0, 1, 2):
            assert 0 <= lib.rs_gated_rec_states_floats(code, B, T, D) <= B * T * D
            assert lib.rs_gated_rec_workspace_floats(code, B, T, D) >= 0
    assert lib.rs_gated_rec_states_floats(0, -1, 5, 5) == 0
    assert lib.rs_gated_rec_states_floats(7, 1, 5, 5) == 0
    assert lib.rs_layernorm_bwd_workspace_floats(-1, 5) == 0


@pytest.mark.parametrize("size, code", [(4, 0), (2, 1), (2, 2)])
def test_recurrence_forms_are_those_named(size, code):
    """The shapes that the kernels are tested with take the forms they are listed for: the queries give
    the tiles and the cut.  One tile keeps no states (narrow long rows excepted); wide and long tiles are
    then told apart by a longer history of the same batch and width."""
    lib = _lib.load()

    def tiles(B, T, D):
        return lib.rs_gated_rec_states_floats(code, B, T, D) / (B * D)
    for form, width, kind, B, T, D in FORMS[size]:
        shape, n = (form, B, T, D), -(-T // STEPS[form])
        assert (width == "part") == (D * size % 8 != 0), shape
        assert (lib.rs_gated_rec_workspace_floats(code, B, T, D) > 0) == (kind == "cut"), shape
        assert (n > 1) == (kind != "one"), shape
        assert tiles(B, T, D) == (n if n > 1 or form == "slim_long" else 0), shape
        if n == 1 and form in ("long", "wide"):
            assert tiles(B, 1025, D) == -(-1025 // STEPS[form]), shape
        if form in ("slim", "wave"):       # of the same length
            assert (D * size <= 64) == (form == "slim"), shape
    for form in STEPS:
        for width in ("-", "part"):
            kinds = {"flat": {"many"}, "short": {"one"}, "wave": {"one", "many"}, "slim": {"many"},
                     "slim_long": {"many", "cut"}}.get(form, {"one", "many", "cut"})
            assert {k for f, w, k, *_ in FORMS[size] if (f, w) == (form, width)} == kinds


def test_size_queries_of_empty_batches():
    """No sequence needs no state and no workspace, whatever the length and the width's form."""
    lib = _lib.load()
    for T in (0, 1, 9, 65, 129, 300, 2000, 5000, 1 << 20):
        for D in (1, 8, 24, 128, 264, 1024, 5000):
            for code in (0, 1, 2):
                assert lib.rs_gated_rec_states_floats(code, 0, T, D) == 0
                assert lib.rs_gated_rec_workspace_floats(code, 0, T, D) == 0


def test_meta_shapes():
    m = dict(device="meta")
    x, p = E(4, 5, 300, dtype=BF16, **m), E(300, **m)
    y, stats = torch.ops.ctr.layer_norm(x, p, p, 1e-5)
    assert y.shape == x.shape and y.dtype == BF16 and stats.shape == (2, 20)
    dx, dparams = torch.ops.ctr.layer_norm_bwd(y, x, p, stats)
    assert dx.shape == x.shape and dparams.shape == (2, 300) and dparams.dtype == F32
    h, last, states = torch.ops.ctr.gated_recurrence(x, None, None, None)
    assert h.shape == (4, 5, 150) and last.shape == (4, 150) and last.dtype == F32
    dv, dgt, dh0 = torch.ops.ctr.gated_recurrence_bwd(h, last, x, None, None, None, states)
    assert dv.shape == x.shape and dgt.numel() == 0 and dh0.shape == (4, 150)
    codes, scales = torch.ops.ctr.pack8(x)
    assert codes.shape == x.shape and codes.dtype == torch.int8 and scales.shape == (4, 5, 3)
    assert torch.ops.ctr.unpack8(codes, scales, F16).dtype == F16


@pytest.fixture
def custom_ops():
    ops.use_custom_ops(True)
    yield
    ops.use_custom_ops(False)


@pytest.mark.parametrize("grad", [False, True])
def test_traced_without_a_device(custom_ops, grad):
    """The functions over fake tensors, with gradients wanted and without (nothing is launched)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(), torch.set_grad_enabled(grad):
        x, p, s = (E(*shape, device="cuda", requires_grad=grad) for shape in ((4, 300, 40), (40,), (4, 40)))
        assert sequence.layer_norm(x, p, p).shape == x.shape
        for g in (x, None):
            h, last = sequence.gated_recurrence(x, g, s if g is not None else None)
            assert h.shape == (4, 300, 40 if g is not None else 20) and last.shape == (4, h.shape[2])
    with FakeTensorMode():
        v, s = E(4, 40, device="cuda", dtype=BF16), E(4, 40, device="cuda")
        h, new = sequence.gated_recurrence_step(v, v, s, s)
        assert new is s and h.shape == v.shape and h.dtype == BF16
        assert sequence.gated_recurrence_step(v)[1].shape == (4, 20)


@pytest.mark.parametrize("save_8bit", [False, True])
def test_encoder_traced_for_serving(custom_ops, save_8bit):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(), torch.no_grad():
        enc = sequence.SequenceEncoder(16, depth=2, save_8bit=save_8bit)
        lengths = E(3, device="cuda", dtype=torch.int64)
        y, states = enc(E(3, 70, 24, device="cuda"), lengths)
        assert y.shape == (3, 70, 24) and states.shape == (2, 3, 16)
        y, states = enc.step(E(3, 24, device="cuda"), states)
        assert y.shape == (3, 24) and states.shape == (2, 3, 16)


def test_step_output_must_not_overlap():
    m = torch.zeros(100)
    state, out = m[:40].view(5, 8), m[8:48].view(5, 8)
    v = E(5, 8)
    for bad in ((out, v, v, state), (state, v, v, out), (out, m[:40].view(5, 8), v, None), (out, v, m[40:80].view(5, 8), None),
                (out, m.view(5, 20)[:, :16], None, None), (out, out.view(5, 8), v, state), (m[39:79].view(5, 8), v, v, state)):
        with pytest.raises(ValueError, match="overlaps"):
            sequence._check_out(*bad)
    for good in ((state, v, v, state), (state.view(5, 8), v, v, state), (m[40:80].view(5, 8), v, v, state),
                 (out, v, v, None), (out, v, v, m[:80].view(5, 16)[:, ::2]), (m[40:40].view(0, 8), m[:0].view(0, 8), v[:0], None),
                 (m[40:80].view(5, 8), m[:40].view(5, 8), m[80:].view(5, 4), None)):
        sequence._check_out(*good)


def test_allocations_are_seen():
    """Outputs and workspaces are made through torch's dispatcher: modes (memory filled in deterministic
    runs, fake tensors, trackers) see them."""
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    with FakeTensorMode():
        t = _lib.empty((2, 3), torch.int8)
    assert isinstance(t, FakeTensor) and t.shape == (2, 3) and t.dtype == torch.int8 and t.is_contiguous()


def test_dense_flag_defaults_off():
    assert not Dense(3).save_8bit and Dense(3, save_8bit=True).save_8bit
    assert packing.scale_shape((2, 129)) == (2, 2)
