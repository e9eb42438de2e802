"""Arguments that ops.group_norm, ops.linear and ops.grouped_linear refuse, before anything reaches a device."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from distributed_machine_learning_amd import _native as N
from distributed_machine_learning_amd import ops

BF = torch.bfloat16


def _t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _norm(x=None, groups=4, **kw):
    return ops.group_norm(_t(2, 3, 3, 16) if x is None else x, groups, **kw)


BUF = torch.zeros(4, 64, dtype=BF)


@pytest.mark.parametrize("error, match, call", [
    (ValueError, "act is one of", lambda: _norm(act="tanh")),
    (ValueError, "act is one of", lambda: _norm(act=None)),
    (TypeError, "x: expected", lambda: _norm(_t(2, 3, 16, dtype=torch.float64))),
    (ValueError, "expected \\[N", lambda: _norm(_t(16))),
    (ValueError, "groups must divide", lambda: _norm(groups=5)),
    (ValueError, "groups must divide", lambda: _norm(groups=0)),
    (ValueError, "groups must divide", lambda: _norm(groups=True)),
    (ValueError, "groups must divide", lambda: _norm(_t(2, 3, 0))),
    (ValueError, "eps", lambda: _norm(eps=-1e-5)),
    (ValueError, "eps", lambda: _norm(eps=float("nan"))),
    (ValueError, "eps", lambda: _norm(eps=1e39)),
    (ValueError, "weight: expected shape", lambda: _norm(weight=_t(8))),
    (TypeError, "bias: expected", lambda: _norm(bias=_t(16, dtype=torch.float16))),
    (ValueError, "last dimension", lambda: _norm(_t(2, 16, 9).transpose(1, 2))),
    (ValueError, "step as one", lambda: _norm(_t(2, 6, 3, 16)[:, ::2, :2])),
    (ValueError, "out: expected", lambda: _norm(out=_t(2, 9, 16))),
    (ValueError, "out: expected", lambda: _norm(out=_t(2, 3, 3, 16, dtype=torch.float32))),
    (ValueError, "overlap each other", lambda: _norm(_t(2, 9, 16), out=_t(2, 1, 16).expand(2, 9, 16))),
    (ValueError, "out overlaps x", lambda: _norm(BUF[:, :16], out=BUF[:, 8:24])),
    (ValueError, "HIP device", lambda: _norm()),
    (ValueError, "HIP device", lambda: _norm(BUF[:, :16], out=BUF[:, 16:32])),  # other columns: no overlap
    (ValueError, "HIP device", lambda: _norm(BUF[:, :16], out=BUF[:, :16])),    # in place
    (ValueError, "no backward", lambda: _norm(weight=torch.ones(16, requires_grad=True))),
])
def test_group_norm_refuses(error, match, call):
    with pytest.raises(error, match=match):
        call()


def _lin(x=None, w=None, **kw):
    return ops.linear(_t(4, 8) if x is None else x, _t(6, 8) if w is None else w, **kw)


@pytest.mark.parametrize("error, match, call", [
    (ValueError, "act is one of", lambda: _lin(act="swish")),
    (TypeError, "x: expected", lambda: _lin(_t(4, 8, dtype=torch.float32))),
    (TypeError, "weight: expected", lambda: _lin(w=_t(6, 8, dtype=torch.float16))),
    (ValueError, "does not fit", lambda: _lin(w=_t(6, 7))),
    (ValueError, "does not fit", lambda: _lin(w=_t(2, 6, 8))),
    (ValueError, "does not fit", lambda: _lin(torch.tensor(1.0, dtype=BF))),
    (ValueError, "last dimension", lambda: _lin(w=_t(8, 6).t())),
    (ValueError, "last dimension", lambda: _lin(_t(8, 4).t())),
    (ValueError, "step as one", lambda: _lin(_t(4, 5, 8)[:, :3])),
    (ValueError, "bias: expected shape", lambda: _lin(bias=_t(5))),
    (TypeError, "bias: expected", lambda: _lin(bias=_t(6, dtype=torch.float16))),
    (TypeError, "out: expected", lambda: _lin(out_dtype=torch.float16)),
    (TypeError, "out is", lambda: _lin(out=_t(4, 6), out_dtype=torch.float32)),
    (ValueError, "out: expected shape", lambda: _lin(out=_t(4, 5))),
    (ValueError, "rows overlap", lambda: _lin(out=_t(1, 6).expand(4, 6))),
    (ValueError, "residual: expected", lambda: _lin(residual=_t(4, 6, dtype=torch.float32))),
    (ValueError, "residual: expected", lambda: _lin(residual=_t(6))),
    (ValueError, "out overlaps x", lambda: _lin(BUF[:, :8], out=BUF[:, 2:8])),
    (ValueError, "out overlaps weight", lambda: _lin(w=BUF[:, :8], out=BUF[:, 4:8])),
    (ValueError, "out overlaps residual", lambda: _lin(residual=BUF[:, 1:7], out=BUF[:, :6])),
    (ValueError, "no backward", lambda: _lin(w=_t(6, 8).requires_grad_())),
    (ValueError, "HIP device", lambda: _lin(residual=BUF[:, :6], out=BUF[:, :6])),
    (ValueError, "HIP device", lambda: _lin(BUF[:, :8], out=BUF[:, 8:14])),
    (ValueError, "different devices", lambda: _lin(bias=torch.zeros(6, device="meta"))),
])
def test_linear_refuses(error, match, call):
    with pytest.raises(error, match=match):
        call()


def _grp(x=None, w=None, ends=None, **kw):
    ends = torch.tensor([1, 4], dtype=torch.int32) if ends is None else ends
    return ops.grouped_linear(_t(4, 8) if x is None else x, _t(2, 6, 8) if w is None else w, ends, **kw)


@pytest.mark.parametrize("error, match, call", [
    (TypeError, "ends: expected", lambda: _grp(ends=torch.tensor([1.0, 4.0]))),
    (ValueError, "contiguous ends", lambda: _grp(ends=torch.tensor([1, 2, 4]))),
    (ValueError, "contiguous ends", lambda: _grp(ends=torch.tensor([1, 0, 4, 0])[::2])),
    (ValueError, "expected x \\[T, K\\]", lambda: _grp(_t(2, 2, 8))),
    (ValueError, "expected x \\[T, K\\]", lambda: _grp(w=_t(6, 8))),
    (ValueError, "does not fit", lambda: _grp(w=_t(2, 6, 7))),
    (ValueError, "bias: expected shape", lambda: _grp(bias=_t(6))),
    (ValueError, "last dimension", lambda: _grp(w=_t(2, 8, 6).transpose(1, 2))),
    (ValueError, "residual: expected", lambda: _grp(residual=_t(3, 6))),
    (ValueError, "out overlaps ends", lambda: (lambda e: _grp(ends=e, out=e.view(BF).as_strided((4, 6), (6, 1))))(
        torch.zeros(32, dtype=torch.int32)[:2].contiguous())),
    (ValueError, "HIP device", lambda: _grp()),
])
def test_grouped_linear_refuses(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_argument_structs_match_the_library():
    """lib() compares the struct sizes; the new ones are among those compared."""
    assert {"GroupNormArgs", "ProductArgs"} <= set(N.ABI_STRUCTS)
    N.lib()


def test_older_library_is_checked_for_the_structs_it_has(monkeypatch):
    """A library from before the last struct loads only where it is asked for by path; a size that differs never does."""
    def library(known, off=0):
        def sizes(out, n):
            for i, name in enumerate(N.ABI_STRUCTS[:known]):
                out[i] = C.sizeof(getattr(N, name)) + off
            return known
        return type("Library", (), {"dml_abi_sizes": staticmethod(sizes)})

    count = len(N.ABI_STRUCTS)
    monkeypatch.delenv("DML_LIB", raising=False)
    N._check_abi(library(count))
    with pytest.raises(N.NativeError):
        N._check_abi(library(count - 1))
    monkeypatch.setenv("DML_LIB", "older.so")
    N._check_abi(library(count - 1))
    with pytest.raises(N.NativeError):
        N._check_abi(library(count - 1, off=8))


def _norm_args(**kw):
    d = {"x": 16, "y": 16, "weight": 0, "bias": 0, "xn": 64, "yn": 64, "ldx": 16, "ldy": 16, "ws": 0, "ws_bytes": 0,
         "N": 1, "HW": 4, "C": 16, "G": 4, "dtype": 0, "act": 0, "eps": 1e-5, **kw}
    return C.byref(N.GroupNormArgs(*d.values()))


@pytest.mark.parametrize("kw", [{"C": 0}, {"G": 0}, {"G": 3}, {"N": -1}, {"HW": -1}, {"dtype": 3}, {"dtype": -1},
                                {"act": 5}, {"act": -1}, {"x": None}, {"y": None}, {"ldy": 15}, {"ldx": -1},
                                {"HW": 2 ** 31 - 1}, {"N": 2 ** 25, "HW": 1, "C": 3, "G": 3}])
def test_library_refuses_group_norm(kw):
    """The library's own checks: nothing is launched, the reason is left for dml_last_error."""
    assert N.lib().dml_group_norm(_norm_args(**kw), None) == -1
    assert N.lib().dml_last_error().startswith(b"dml_group_norm")


def test_library_group_norm_asks_for_its_workspace():
    """A sample too long for one workgroup: the size comes back, and nothing is launched without it."""
    need = N.lib().dml_group_norm(_norm_args(HW=200000, xn=3200000, yn=3200000), None)
    assert need > 0 and need % 8 == 0
    assert N.lib().dml_group_norm(_norm_args(HW=200000, xn=3200000, yn=3200000, ws=16, ws_bytes=need - 1), None) == need
    assert N.lib().dml_group_norm(_norm_args(N=0), None) == 0
    assert N.lib().dml_group_norm(None, None) == -1


def _prod_args(**kw):
    d = {"x": 16, "w": 16, "bias": 0, "res": 0, "y": 16, "ends": 0, "ldx": 8, "ldw": 8, "w_group": 0, "bias_group": 0,
         "ldr": 0, "ldy": 8, "M": 4, "N": 8, "K": 8, "E": 1, "dtype": 0, "out_f32": 0, "act": 0, "act_last": 0,
         "ends64": 0, "fill": 0, **kw}
    return C.byref(N.ProductArgs(*d.values()))


@pytest.mark.parametrize("kw", [{"M": -1}, {"N": -1}, {"K": -1}, {"E": -1}, {"E": 2}, {"K": 2 ** 30 + 1}, {"M": 2 ** 31 - 1},
                                {"dtype": 2}, {"dtype": -1}, {"act": 5}, {"x": None}, {"w": None}, {"y": None}, {"ldy": 7},
                                {"ldx": -1}, {"ldw": -8}, {"ldr": -1}, {"w_group": -1}, {"ldx": 2 ** 62}, {"ldy": 2 ** 62},
                                {"M": 2 ** 31 - 600, "N": 2 ** 20, "ldy": 2 ** 20}])
def test_library_refuses_product(kw):
    assert N.lib().dml_product(_prod_args(**kw), None) == -1
    assert N.lib().dml_last_error().startswith(b"dml_product")


def test_library_product_of_nothing():
    assert N.lib().dml_product(_prod_args(M=0), None) == 0
    assert N.lib().dml_product(_prod_args(N=0), None) == 0
    assert N.lib().dml_product(None, None) == -1


@pytest.mark.parametrize("what, call", [
    ("x", lambda t: ops.linear(t, _t(8, 8), residual=t, out=t)),
    ("x", lambda t: ops.linear(t, _t(8, 8), residual=t, act_last=True, act="relu", out=t)),
    ("weight", lambda t: ops.linear(_t(8, 8), t, residual=t, out=t)),
    ("x", lambda t: ops.grouped_linear(t, _t(2, 8, 8), torch.tensor([1, 8]), residual=t, out=t)),
    ("bias", lambda t: ops.grouped_linear(_t(8, 8), _t(8, 8, 8), torch.arange(8), bias=t, residual=t, out=t)),
    ("weight", lambda t: ops.group_norm(t[0].view(1, 1, 8), 4, weight=t[0], out=t[0].view(1, 1, 8))),
])
def test_out_that_is_the_residual_and_another_operand_too(what, call):
    """One tensor in two places: x and weight are read by many workgroups, so out is refused, object or view alike."""
    with pytest.raises(ValueError, match=f"out overlaps {what}"):
        call(_t(8, 8))


@pytest.mark.parametrize("shape, strides, fits", [
    ((4, 9, 16), (16, 16, 1), False),    # windows over one sequence: samples share eight of nine positions
    ((2, 9, 16), (143, 16, 1), False),   # by one element
    ((2, 9, 16), (144, 16, 1), True),
    ((2, 9, 16), (16, 32, 1), True),     # samples between the positions of the first
    ((3, 9, 16), (16, 32, 1), False),
    ((3, 9, 16), (20, 56, 1), True),
    ((3, 9, 16), (20, 55, 1), False),
    ((2, 1, 16), (16, 1, 1), True),
    ((2, 1, 16), (15, 1, 1), False),
    ((2, 2, 3, 16), (40, 48, 16, 1), False),
    ((1, 9, 16), (1, 16, 1), True),
])
def test_group_norm_out_that_overlaps_itself(shape, strides, fits):
    out = torch.zeros(2000, dtype=BF).as_strided(shape, strides)
    with pytest.raises(ValueError, match="HIP device" if fits else "overlap each other"):
        ops.group_norm(_t(*shape), 4, out=out)


@pytest.mark.parametrize("steps, other, fits", [
    ((96, 32), 16, True), ((128, 32), 16, True), ((112, 32), 16, True),
    ((80, 32), 16, False),                       # the second sample of x begins where out's third position lies
    ((95, 32), 16, False),
    ((110, 40), 24, False), ((110, 40), 16, False), ((112, 40), 16, True), ((120, 40), 24, True), ((120, 40), 25, False),
    ((120, 40), 15, False), ((120, 40), -16, True), ((120, 40), -24, True), ((120, 40), -25, False), ((120, 40), 40, False),
    ((32, 64), 16, True), ((31, 64), 16, False), ((32, 63), 16, False),  # samples between the positions of the first
])
def test_group_norm_out_in_other_columns(steps, other, fits):
    """Other columns of the same rows, by x's strides."""
    buf = torch.zeros(500, dtype=BF)
    shape = (2, 3, 16)
    x, out = (buf.as_strided(shape, (*steps, 1), at) for at in (40, 40 + other))
    mine, theirs = (set((torch.arange(500).as_strided(shape, (*steps, 1), at)).flatten().tolist()) for at in (40, 40 + other))
    assert fits == (not mine & theirs)
    with pytest.raises(ValueError, match="HIP device" if fits else "out overlaps x"):
        ops.group_norm(x, 4, out=out)


@pytest.mark.parametrize("no_grad", (False, True))
@pytest.mark.parametrize("call", [
    lambda d: _norm(d(_t(2, 3, 3, 16))), lambda d: _norm(weight=d(_t(16))), lambda d: _norm(bias=d(_t(16))),
    lambda d: _norm(out=d(_t(2, 3, 3, 16))), lambda d: _lin(d(_t(4, 8))), lambda d: _lin(w=d(_t(6, 8))),
    lambda d: _lin(bias=d(_t(6))), lambda d: _lin(residual=d(_t(4, 6))), lambda d: _grp(d(_t(4, 8))), lambda d: _grp(w=d(_t(2, 6, 8))),
])
def test_forward_mode_tangents_are_refused(call, no_grad):
    """Results without the tangent would be wrong derivatives, with no error; tensors without one pass in a dual level."""
    with torch.set_grad_enabled(not no_grad), forward_ad.dual_level():
        with pytest.raises(ValueError, match="no derivative"):
            call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError, match="HIP device"):
            call(lambda t: t)


def test_forward_mode_through_a_function_transform():
    with pytest.raises(ValueError, match="no derivative"):
        torch.func.jvp(lambda t: _norm(t), (_t(2, 3, 3, 16),), (_t(2, 3, 3, 16),))


def _merged(x, groups, rows, between=True, lost=None, last_full=False):
    """Group norm from chunks of `rows` positions, merged in fp32, or with a mistake in the merge."""
    n, c = x.shape[0], x.shape[-1]
    v = x.float().reshape(n, -1, groups, c // groups)
    chunks = [p for i, p in enumerate(v.split(rows, 1)) if i != lost]
    mean = torch.stack([p.mean((1, 3)) for p in chunks])
    m2 = torch.stack([(p - p.mean((1, 3), keepdim=True)).square().sum((1, 3)) for p in chunks])
    size = torch.tensor([rows if last_full else p.shape[1] for p in chunks]).float()[:, None, None] * (c // groups)
    mu = (mean * size).sum(0) / size.sum()
    var = (m2 + (size * (mean - mu).square() if between else 0)).sum(0) / size.sum()
    return ((v - mu[:, None, :, None]) / torch.sqrt(var + 1e-5)[:, None, :, None]).reshape(x.shape).to(x.dtype)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("drift", ("ramp", "steps"))
def test_the_tolerance_of_merged_chunks_tells_mistakes(drift, dtype):
    """The bound that the kernels' merged chunks are held to accepts a right merge, and no missing term or chunk."""
    from test_layers_edges_gpu import drifting, steps_of_chunks, tight64
    from test_layers_gpu import close

    x = (torch.randn(1, 9000, 48, generator=torch.Generator().manual_seed(3)) + drifting(drift, 9000, "cpu")).to(dtype)
    y, err = tight64(x, 3, steps_of_chunks())
    close(_merged(x, 3, 512), y, err)
    for mistake in ({"between": False}, {"lost": 7}, {"lost": 17}, {"last_full": True}):
        with pytest.raises(AssertionError, match="times the tolerance"):
            close(_merged(x, 3, 512, **mistake), y, err)
