"""Arrays that overlap are refused before anything is launched; arrays that only interleave are not.  No GPU needed: the calls are
refused, or run on the kernels' host build."""
import ctypes as C

import numpy as np
import pytest

from test_sequence_kernels_cpu import sim  # noqa: F401

capi = pytest.importorskip("mfcc_amd._capi")
R = capi.MfccRows
FAR = 1 << 30     # addresses are never dereferenced: every call is refused


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def scan(lib, x, g, y, n=2, steps=10, h0=None, last=None, ckpt=None, ws=None, dtype=0):
    return lib.mfcc_gated_scan(None, n, steps, 8, dtype, 0, 0, x, g, h0, y, last, ckpt, ws, None)


def backward(lib, gx, gg, gh0=None, x=None, ckpt=8 * FAR, gy=None, gl=None):
    return lib.mfcc_gated_scan_backward(None, 2, 10, 8, 0, 0, 0, x or R(FAR, 80, 8), R(2 * FAR, 80, 8), ckpt, gy, gl, gx, gg, gh0, None, None)


def norm(lib, x, y, state_in=None, state_out=None, dtype=0):
    return lib.mfcc_running_norm(None, 2, 10, 8, 0.9, 1e-5, 0, x, state_in, y, dtype, state_out, None, None)


def drop(lib, x, y, step=None, per=0):
    return lib.mfcc_feature_dropout(None, 2, 10, 8, 0, per, 100, 1, 0, step, x, y, None)


def step(lib, x=FAR, g=2 * FAR, si=3 * FAR, so=4 * FAR, y=5 * FAR, dtype=0, x_ld=8, y_ld=8):
    return lib.mfcc_gated_scan_step(4, 8, dtype, 0, x, x_ld, g, 8, si, so, y, y_ld, None)


A, B, Y = R(FAR, 80, 8), R(2 * FAR, 80, 8), R(3 * FAR, 80, 8)    # [2, 10, 8] float32: 640 bytes each


@pytest.mark.parametrize("call", [
    lambda l: scan(l, A, B, R(FAR + 32, 80, 8)), lambda l: scan(l, A, B, R(FAR - 32, 80, 8)),               # shifted by a row
    lambda l: scan(l, A, B, R(2 * FAR + 4, 80, 8)), lambda l: scan(l, A, B, R(FAR, 8, 16)),                 # by an element; the other order
    lambda l: scan(l, A, B, R(FAR + 636, 80, 8)), lambda l: scan(l, A, B, R(FAR - 636, 80, 8)),             # by all but an element
    lambda l: scan(l, R(FAR, 160, 16), B, R(FAR + 28, 160, 16)), lambda l: scan(l, R(FAR, 160, 16), B, R(FAR + 36, 160, 16)),
    lambda l: scan(l, R(FAR, 0, 0), B, R(FAR, 80, 8)),                                                       # one row for all, under y
    lambda l: scan(l, A, B, Y, h0=3 * FAR + 100), lambda l: scan(l, A, B, Y, last=FAR), lambda l: scan(l, A, B, Y, last=3 * FAR + 636),
    lambda l: scan(l, A, B, Y, h0=5 * FAR, last=5 * FAR), lambda l: scan(l, A, B, Y, h0=5 * FAR, last=5 * FAR + 60),
    lambda l: scan(l, A, B, Y, ckpt=FAR), lambda l: scan(l, A, B, Y, last=5 * FAR, ckpt=5 * FAR + 32),
    lambda l: scan(l, R(FAR, 0, 8), R(2 * FAR, 0, 8), R(3 * FAR, 0, 8), n=1, steps=1 << 20, ws=2 * FAR + 16),
    lambda l: backward(l, A, Y), lambda l: backward(l, Y, R(2 * FAR, 80, 8)), lambda l: backward(l, Y, Y), lambda l: backward(l, Y, R(5 * FAR, 80, 8), gh0=3 * FAR),
    lambda l: backward(l, Y, R(5 * FAR, 80, 8), gy=R(5 * FAR, 80, 8)), lambda l: backward(l, Y, R(5 * FAR, 80, 8), gl=6 * FAR, gh0=6 * FAR + 4),
    lambda l: norm(l, A, R(FAR + 32, 80, 8)), lambda l: norm(l, A, R(FAR, 80, 8), dtype=1), lambda l: norm(l, A, A, state_in=FAR + 600),
    lambda l: norm(l, A, Y, state_out=FAR), lambda l: norm(l, A, Y, state_in=5 * FAR, state_out=5 * FAR),
    lambda l: norm(l, A, Y, state_in=5 * FAR, state_out=5 * FAR + 68), lambda l: norm(l, A, Y, state_in=5 * FAR + 132, state_out=5 * FAR),
    lambda l: drop(l, A, R(FAR + 32, 80, 8)), lambda l: drop(l, A, R(FAR, 88, 8)), lambda l: drop(l, A, R(FAR + 4, 80, 8), per=1),
    lambda l: drop(l, A, Y, step=3 * FAR + 8), lambda l: drop(l, A, Y, step=3 * FAR - 4, per=2),
    lambda l: step(l, y=FAR + 32), lambda l: step(l, y=3 * FAR + 4), lambda l: step(l, so=3 * FAR + 32), lambda l: step(l, so=3 * FAR - 32),
    lambda l: step(l, y=FAR, x_ld=16), lambda l: step(l, dtype=1, y=4 * FAR), lambda l: step(l, so=FAR + 4),
    lambda l: scan(l, R(FAR, 80, (1 << 56) + 1), B, Y), lambda l: step(l, x_ld=(1 << 56) + 1)])
def test_overlap_is_refused(lib, call):
    assert call(lib) == capi.ERR_INVALID
    assert b"overlap" in lib.mfcc_last_error() or b"2^56" in lib.mfcc_last_error() or b"shape" in lib.mfcc_last_error()


def view(buf, at, ss, rs):
    return R(buf.ctypes.data + 4 * at, ss, rs), np.lib.stride_tricks.as_strided(buf[at:], (2, 10, 8), (4 * ss, 4 * rs, 4))


@pytest.mark.parametrize("where", [
    [(0, 80, 8), (160, 80, 8), (320, 80, 8)],        # one after the other
    [(0, 240, 24), (8, 240, 24), (16, 240, 24)],     # columns of wider rows
    [(0, 240, 8), (80, 240, 8), (160, 240, 8)],      # parts of longer sequences
    [(0, 8, 48), (16, 8, 48), (32, 8, 48)],          # time-major, parts of a longer list of sequences
    [(0, 240, 24), (8, 240, 24), (8, 240, 24)],      # y over the gates, x between their rows
    [(0, 80, 8), (160, 80, 8), (0, 80, 8)],          # in place
    [(0, 160, 16), (8, 160, 16), (320, 8, 16)],      # y in another order
    [(0, 0, 0), (8, 0, 8), (160, 80, 8)]])           # inputs of one row, of one sequence
def test_interleaved_arrays_are_taken(sim, where):
    """Three views of one buffer; the surroundings stay as they were."""
    buf = np.random.default_rng(1).uniform(-0.9, 0.9, 1000).astype(np.float32)
    (x, xv), (g, gv), (y, yv) = (view(buf, *w) for w in where)
    xs, gs, h = xv.astype(np.float64), gv.astype(np.float64), np.zeros((2, 8))
    want = np.zeros((2, 10, 8))
    for t in range(10):
        want[:, t] = h = gs[:, t] * h + xs[:, t]
    mask = np.zeros(1000, bool)
    np.lib.stride_tricks.as_strided(mask[where[2][0]:], (2, 10, 8), (where[2][1], where[2][2], 1))[:] = True
    before = buf.copy()
    assert sim.mfcc_gated_scan(None, 2, 10, 8, 0, 0, 0, x, g, None, y, None, None, None, None) == 0
    # gates below 0.9: a memory of ten rows, each rounding twice
    assert np.abs(yv - want).max() <= 16 * 2.0 ** -24 * 11 * 10
    assert np.array_equal(buf[~mask], before[~mask])


def test_step_in_place(sim):
    """Any of the arrays of a step may be one and the same."""
    rng = np.random.default_rng(2)
    for out, state_out in ((0, 2), (1, 2), (2, 2), (3, 2), (3, 0), (0, 4), (4, 4)):
        a = [rng.uniform(-1, 1, (4, 8)).astype(np.float32) for _ in range(5)]
        want = a[1].astype(np.float64) * a[2] + a[0]
        p = [C.c_void_p(t.ctypes.data) for t in a]
        assert sim.mfcc_gated_scan_step(4, 8, 0, 0, p[0], 8, p[1], 8, p[2], p[state_out], p[out], 8, None) == 0
        for k in (out, state_out):
            assert np.abs(a[k] - want).max() <= 2 * 2.0 ** -24 * 2
