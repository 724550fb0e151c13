"""Refusals of the channels-last operators' calls (no GPU needed: nothing gets as far as a launch)."""
from __future__ import annotations

import ctypes

import pytest

import s2b200

torch = pytest.importorskip("torch")

BASE = 1 << 20  # an address that is never read


def _norm(**kw):
    d = dict(samples=2, channels=64, groups=32, activation=2, positions=100, in_dtype=s2b200.S2_F16,
             out_dtype=s2b200.S2_F16, eps=1e-6, x=BASE, x_row=64, x_sample=6400, weight=None, bias=None, y=2 * BASE,
             y_row=64, y_sample=6400, workspace=4 * BASE, workspace_bytes=1 << 30, err=None)
    d.update(kw)
    return s2b200.GroupNormActDesc(**d)


def _linear(**kw):
    d = dict(N=64, K=128, activation=0, dtype=s2b200.S2_F16, out_dtype=s2b200.S2_F16, M=10, x=BASE, ldx=128,
             w=2 * BASE, ldw=128, bias=None, residual=None, ldr=0, y=3 * BASE, ldy=64, workspace=4 * BASE,
             workspace_bytes=1 << 30, err=None)
    d.update(kw)
    return s2b200.LinearActDesc(**d)


def _call(fn, desc):
    launches = ctypes.c_int(-1)
    status = getattr(s2b200.lib(), fn)(None, ctypes.byref(desc), ctypes.byref(launches))
    return status, launches.value


INVALID, UNSUPPORTED = s2b200.S2_INVALID_ARGUMENT, s2b200.S2_UNSUPPORTED

NORM_REFUSALS = [
    (dict(samples=-1), INVALID), (dict(positions=-1), INVALID), (dict(channels=0), INVALID), (dict(groups=0), INVALID),
    (dict(groups=33), INVALID), (dict(x=None), INVALID), (dict(y=None), INVALID), (dict(x=BASE + 1), INVALID),
    (dict(y=2 * BASE + 1), INVALID), (dict(weight=BASE + 2), INVALID), (dict(bias=BASE + 2), INVALID),
    (dict(x_row=63), INVALID), (dict(y_row=63), INVALID), (dict(x_sample=6399), INVALID), (dict(x_sample=0), INVALID),
    (dict(y_sample=6399), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID),
    (dict(eps=float("inf")), INVALID), (dict(activation=5), UNSUPPORTED), (dict(activation=-1), UNSUPPORTED),
    (dict(in_dtype=7), UNSUPPORTED), (dict(out_dtype=s2b200.S2_BF16), UNSUPPORTED),
    (dict(out_dtype=s2b200.S2_F32), UNSUPPORTED), (dict(channels=4096, groups=2048, x_row=4096, y_row=4096), UNSUPPORTED),
    (dict(samples=1 << 20), UNSUPPORTED), (dict(y=BASE + 64), INVALID), (dict(y=BASE, y_row=72, y_sample=7200), INVALID),
    (dict(y=BASE, in_dtype=s2b200.S2_F32), INVALID), (dict(x_row=1 << 50, x_sample=1 << 60), INVALID),
    (dict(x_row=80, y_row=80, x_sample=8000, y_sample=8000, y=BASE + 32), INVALID),
    (dict(positions=1 << 41), UNSUPPORTED), (dict(x_sample=1 << 62), INVALID), (dict(y_sample=1 << 62), INVALID),
    (dict(positions=1 << 31, x_row=1 << 40), INVALID), (dict(positions=1 << 31, y_row=1 << 40), INVALID),
    (dict(positions=1 << 31, channels=1 << 30, x_row=1 << 30, y_row=1 << 30), UNSUPPORTED),
]


@pytest.mark.parametrize("kw,status", NORM_REFUSALS, ids=lambda v: str(v))
def test_norm_refusals(kw, status):
    assert _call("s2_group_norm_act", _norm(**kw)) == (status, 0)
    assert "group_norm_act" in s2b200.last_error()


@pytest.mark.parametrize("kw", [dict(workspace=None), dict(workspace_bytes=0), dict(workspace=4 * BASE + 4)], ids=str)
def test_norm_workspace_refusals(kw):
    big = dict(positions=1 << 22, x_sample=1 << 28, y_sample=1 << 28, y=1 << 40)
    if s2b200.lib().s2_group_norm_act_workspace_bytes(ctypes.byref(_norm(**big))) == 0:
        pytest.skip("this size needs no workspace")
    assert _call("s2_group_norm_act", _norm(**big, **kw)) == (INVALID, 0)


@pytest.mark.parametrize("kw", [dict(samples=0), dict(positions=0)], ids=str)
def test_norm_of_nothing(kw):
    assert _call("s2_group_norm_act", _norm(x=None, y=None, workspace=None, **kw)) == (0, 0)
    assert s2b200.lib().s2_group_norm_act_workspace_bytes(ctypes.byref(_norm(**kw))) == 0


LINEAR_REFUSALS = [
    (dict(M=-1), INVALID), (dict(N=0), INVALID), (dict(K=0), INVALID), (dict(x=None), INVALID), (dict(w=None), INVALID),
    (dict(y=None), INVALID), (dict(x=BASE + 1), INVALID), (dict(w=BASE + 1), INVALID), (dict(y=BASE + 1), INVALID),
    (dict(bias=BASE + 2), INVALID), (dict(residual=5 * BASE + 1, ldr=64), INVALID), (dict(ldx=127), INVALID),
    (dict(ldw=127), INVALID), (dict(ldy=63), INVALID), (dict(residual=5 * BASE, ldr=63), INVALID),
    (dict(activation=5), UNSUPPORTED), (dict(dtype=s2b200.S2_F32, out_dtype=s2b200.S2_F32), UNSUPPORTED),
    (dict(out_dtype=s2b200.S2_BF16), UNSUPPORTED), (dict(M=1 << 31), UNSUPPORTED), (dict(N=1 << 22, ldy=1 << 22), UNSUPPORTED),
    (dict(K=1 << 22, ldx=1 << 22, ldw=1 << 22), UNSUPPORTED), (dict(y=BASE), INVALID), (dict(y=2 * BASE + 256), INVALID),
    (dict(residual=3 * BASE, ldr=72), INVALID), (dict(residual=3 * BASE + 2, ldr=64), INVALID),
    (dict(bias=3 * BASE + 1024), INVALID), (dict(ldx=1 << 50), INVALID),
    (dict(out_dtype=s2b200.S2_F32, y=3 * BASE + 2), INVALID),
]


@pytest.mark.parametrize("kw,status", LINEAR_REFUSALS, ids=lambda v: str(v))
def test_linear_refusals(kw, status):
    assert _call("s2_linear_act", _linear(**kw)) == (status, 0)
    assert "linear_act" in s2b200.last_error()


def test_linear_of_no_rows():
    assert _call("s2_linear_act", _linear(M=0, x=None, y=None, workspace=None)) == (0, 0)
    assert s2b200.lib().s2_linear_act_workspace_bytes(ctypes.byref(_linear(M=0))) == 0


def test_null_descriptions():
    for fn in ("s2_group_norm_act", "s2_linear_act"):
        assert getattr(s2b200.lib(), fn)(None, None, None) == INVALID
        assert getattr(s2b200.lib(), fn + "_workspace_bytes")(None) == 0


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(4, 64, dtype=torch.float16)
    for call in (lambda: s2b200.group_norm_act(x, 8), lambda: s2b200.linear_act(x, x)):
        with pytest.raises(s2b200.S2Error) as e:
            call()
        assert e.value.status == INVALID


def test_packed_descriptions_match_the_structures():
    """The wrappers pack their descriptions with struct; the layouts are the structures'."""
    for layout, cls in ((s2b200._NORM_LAYOUT, s2b200.GroupNormActDesc), (s2b200._LINEAR_LAYOUT, s2b200.LinearActDesc)):
        assert layout.size == ctypes.sizeof(cls)
        names = [n for n, _ in cls._fields_]
        got = cls.from_buffer_copy(layout.pack(*range(1, len(names) + 1)))
        assert [int(getattr(got, n)) for n in names] == list(range(1, len(names) + 1))


def test_device_error_without_a_device():
    """Asked where no device can answer: an error, not a code."""
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    code = ctypes.c_int32(7)
    assert s2b200.lib().s2_operator_device_error(ctypes.byref(code)) == s2b200.S2_INFERENCE_FAILED and code.value == 0
    assert s2b200.lib().s2_operator_device_error(None) == s2b200.S2_INFERENCE_FAILED


EMPTY = [(0, 64), (3, 0, 64), (0, 3, 64), (2, 3, 0, 64), (2, 0, 3, 64), (2, 0, 0, 64)]


@pytest.mark.parametrize("shape", EMPTY, ids=str)
def test_pitch_of_no_rows(shape):
    assert s2b200._pitch(torch.empty(shape), 0, "x")[0] == 0
    assert s2b200._pitch(torch.empty((5,) + shape), 1, "x")[0] == 0
    assert s2b200._pitch(torch.empty(shape[:-1] + (128,))[..., ::2], 0, "x")[0] == 0


@pytest.mark.parametrize("at,value", [(2, 1 << 40), (2, 8.0), (0, 1 << 31), (1, -(1 << 40)), (7, None), (7, "1")],
                         ids=str)
def test_numbers_that_fit_no_description(at, value):
    values = [2, 64, 32, 0, 100, 1, 1, 1e-6, BASE, 64, 6400, 0, 0, 2 * BASE, 64, 6400, 0, 0, 0]
    values[at] = value
    with pytest.raises(s2b200.S2Error) as e:
        s2b200._pack(s2b200._NORM_LAYOUT, *values)
    assert e.value.status == INVALID


# large enough for a workspace (slices of a grid)
LARGE = dict(samples=4, channels=512, positions=1 << 14, x_row=512, y_row=512, x_sample=1 << 23, y_sample=1 << 23, x=1 << 32,
             y=2 << 32, weight=3 << 32, bias=4 << 32, workspace=5 << 32)


@pytest.mark.parametrize("kw", [dict(weight=2 << 32), dict(bias=2 << 32), dict(weight=(2 << 32) - 2044),
                                dict(bias=(2 << 32) + (4 << 24) - 4), dict(workspace=1 << 32), dict(workspace=(2 << 32) + 4096),
                                dict(workspace=(1 << 32) - 16), dict(workspace=(3 << 32) + 2032), dict(workspace=(4 << 32) - 16)], ids=str)
def test_norm_refuses_what_would_be_overwritten(kw):
    d = _norm(**(LARGE | kw))
    assert s2b200.lib().s2_group_norm_act_workspace_bytes(ctypes.byref(d)) > 0
    assert _call("s2_group_norm_act", d) == (INVALID, 0)
    assert "overlaps" in s2b200.last_error()


@pytest.mark.parametrize("at", [BASE, BASE + 2048, 2 * BASE, 3 * BASE, 5 * BASE + 240, 6 * BASE - 2096], ids=str)
def test_linear_refuses_a_workspace_on_its_operands(at):
    """x in rows of 129 values is packed into the workspace."""
    d = _linear(ldx=129, workspace=at, bias=5 * BASE, residual=6 * BASE, ldr=64)
    assert s2b200.lib().s2_linear_act_workspace_bytes(ctypes.byref(d)) == 10 * 128 * 2
    assert _call("s2_linear_act", d) == (INVALID, 0)
    assert "workspace overlaps" in s2b200.last_error()


@pytest.mark.parametrize("pad,dtype", [(3, s2b200.S2_F16), (1, s2b200.S2_F32)], ids=str)
def test_norm_takes_wide_rows_in_slices_that_a_block_holds(pad, dtype):
    """Rows not on 16 bytes are read value by value, a column a thread: 512 channels are two slices of 256 columns, which
    blocks hold, like twice as many samples of 256 channels."""
    def workspace(samples, channels, groups):
        row = channels + pad
        d = _norm(samples=samples, channels=channels, groups=groups, positions=14400, x_row=row, y_row=row,
                  x_sample=14400 * row, y_sample=14400 * row, in_dtype=dtype, out_dtype=dtype, y=1 << 40)
        return s2b200.lib().s2_group_norm_act_workspace_bytes(ctypes.byref(d))
    assert workspace(6, 512, 32) == workspace(12, 256, 16) > 0


def test_linear_looks_at_the_residuals_pitch_only_with_a_residual():
    """Past the checks of pitches, to the last one: y on its bias."""
    for ldr in (1 << 50, -1, 0):
        assert _call("s2_linear_act", _linear(ldr=ldr, bias=3 * BASE)) == (INVALID, 0)
        assert "y overlaps" in s2b200.last_error()
    assert _call("s2_linear_act", _linear(ldr=1 << 50, residual=6 * BASE, bias=3 * BASE)) == (INVALID, 0)
    assert "pitch" in s2b200.last_error()


@pytest.mark.parametrize("channels,groups", [(1 << 30, 1), ((1 << 31) - 4, 1), ((1 << 31) - 1024, 1024), ((1 << 31) - 1, 1)], ids=str)
def test_norm_of_as_many_channels_as_an_int_holds(channels, groups):
    """Planned without overflow: to the last check, y on x."""
    for dtype in (s2b200.S2_F32, s2b200.S2_BF16):
        d = _norm(samples=1, positions=1000, channels=channels, groups=groups, x_row=channels, y_row=channels, in_dtype=dtype,
                  out_dtype=dtype, y=BASE + 64)
        s2b200.lib().s2_group_norm_act_workspace_bytes(ctypes.byref(d))
        assert s2b200.last_error() == ""
        assert _call("s2_group_norm_act", d) == (INVALID, 0)
        assert "overlaps" in s2b200.last_error()


def test_operands_between_the_rows_of_y():
    """Weights in the gaps of y's pitched rows overlap nothing; a byte further they do. (The calls end at the missing
    workspace.)"""
    row = 512 + 2048
    d = LARGE | dict(y_row=row, y_sample=(1 << 14) * row, workspace=None)
    for at, what in ((1024, "workspace of"), (7 * 2 * row + 1024, "workspace of"), (7 * 2 * row + 2 * row - 2048, "workspace of"),
                     (1020, "overlaps"), (7 * 2 * row + 2 * row - 2044, "overlaps")):
        for name in ("weight", "bias"):
            assert _call("s2_group_norm_act", _norm(**(d | {name: d["y"] + at}))) == (INVALID, 0)
            assert what in s2b200.last_error(), (at, name)
