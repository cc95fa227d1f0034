"""Refusals of the operators along time that need no GPU: the C entry points turn bad arguments into
error codes before anything is launched, the Python wrappers into ValueErrors."""
import ctypes as C

import pytest
import torch

capi = pytest.importorskip("mfcc_amd._capi")


@pytest.fixture(scope="module")
def lib():
    return capi.load()


P = C.c_void_p(4096)     # never dereferenced: every call below is refused


def rows(ss=0, rs=8, p=4096):
    return capi.MfccRows(p, ss, rs)


def scan(lib, n=1, steps=10, ncol=8, dtype=0, form=0, x=None, g=None, y=None):
    return lib.mfcc_gated_scan(None, n, steps, ncol, dtype, form, 0, x or rows(), g or rows(), None, y or rows(), None, None, None, None)


def backward(lib, n=1, steps=10, ckpt=P, gy=None, gx=None, gg=None):
    return lib.mfcc_gated_scan_backward(None, n, steps, 8, 0, 0, 0, rows(), rows(), ckpt, gy, None, gx or rows(), gg or rows(), None, None, None)


def norm(lib, n=1, steps=10, ncol=8, decay=0.9, eps=1e-5, x=None, y=None, dtype=0, state_in=None, state_out=None):
    return lib.mfcc_running_norm(None, n, steps, ncol, decay, eps, 0, x or rows(), state_in, y or rows(), dtype, state_out, None, None)


def drop(lib, n=1, steps=10, ncol=8, dtype=0, per=0, thr=100, x=None, y=None):
    return lib.mfcc_feature_dropout(None, n, steps, ncol, dtype, per, thr, 1, 0, None, x or rows(), y or rows(), None)


def step(lib, n=4, ncol=8, dtype=0, form=0, x_ld=8, y_ld=8, x=P):
    return lib.mfcc_gated_scan_step(n, ncol, dtype, form, x, x_ld, P, 8, P, P, P, y_ld, None)


@pytest.mark.parametrize("call", [
    lambda l: scan(l, ncol=0), lambda l: scan(l, ncol=(1 << 20) + 1), lambda l: scan(l, n=-1), lambda l: scan(l, steps=-1),
    lambda l: scan(l, steps=1 << 31), lambda l: scan(l, dtype=3), lambda l: scan(l, dtype=-1), lambda l: scan(l, form=2),
    lambda l: scan(l, x=rows(p=0)), lambda l: scan(l, g=rows(p=0)), lambda l: scan(l, y=rows(p=0)), lambda l: scan(l, x=rows(rs=-8)),
    lambda l: scan(l, y=rows(rs=7)), lambda l: scan(l, n=2, y=rows(ss=79)), lambda l: scan(l, n=2, y=rows(ss=8, rs=15)),
    lambda l: backward(l, ckpt=None), lambda l: backward(l, gx=rows(rs=4)), lambda l: backward(l, gg=rows(p=0)),
    lambda l: backward(l, gy=rows(rs=-1)),
    lambda l: norm(l, decay=0.0), lambda l: norm(l, decay=1.5), lambda l: norm(l, decay=float("nan")), lambda l: norm(l, eps=-1.0),
    lambda l: norm(l, eps=float("nan")), lambda l: norm(l, dtype=7), lambda l: norm(l, y=rows(rs=1)), lambda l: norm(l, state_in=P, state_out=P),
    lambda l: drop(l, per=3), lambda l: drop(l, thr=-1), lambda l: drop(l, thr=65537), lambda l: drop(l, dtype=9), lambda l: drop(l, y=rows(rs=2)),
    lambda l: step(l, ncol=0), lambda l: step(l, dtype=5), lambda l: step(l, form=9), lambda l: step(l, y_ld=7), lambda l: step(l, x_ld=-1),
    lambda l: step(l, x=None)])
def test_bad_arguments_are_refused(lib, call):
    assert call(lib) == capi.ERR_INVALID
    assert lib.mfcc_last_error()


def test_nothing_to_do_is_no_error(lib):
    assert scan(lib, n=0) == 0 and norm(lib, n=0) == 0 and drop(lib, steps=0) == 0 and step(lib, n=0) == 0 and backward(lib, n=0) == 0


def test_sizes(lib):
    """Checkpoints and workspace: never negative for valid shapes, an error code for the others."""
    for n, steps, ncol in ((0, 5, 3), (1, 0, 3), (1, 1, 1), (32, 700, 512), (1, 360000, 39), (10000, 299, 39)):
        for dtype in range(3):
            assert lib.mfcc_gated_scan_checkpoints(None, n, steps, ncol, dtype) >= (n * ncol if steps else 0)
            assert lib.mfcc_sequence_workspace(None, n, steps, ncol, dtype) >= 0
    assert lib.mfcc_gated_scan_checkpoints(None, 1, 1, 0, 0) == capi.ERR_INVALID
    assert lib.mfcc_sequence_workspace(None, 1, -1, 4, 0) == capi.ERR_INVALID
    assert lib.mfcc_sequence_workspace(None, 1, 1, 4, 3) == capi.ERR_INVALID


def test_host_tensors_are_refused():
    import mfcc_amd
    x = torch.zeros(4, 8)
    for f in (lambda: mfcc_amd.gated_scan(x, x), lambda: mfcc_amd.gated_scan_step(x, x, x), lambda: mfcc_amd.running_norm(x),
              lambda: mfcc_amd.feature_dropout(x, 0.5, 1)):
        with pytest.raises(ValueError):
            f()
    sums = torch.tensor([4.0, 8.0, 20.0], dtype=torch.float64)
    assert mfcc_amd.running_norm_state(sums, 10.0, 2).tolist() == [[10.0, 2.0, 10.0]] * 2
    for bad in (sums.float(), sums[:2]):
        with pytest.raises(ValueError):
            mfcc_amd.running_norm_state(bad, 1.0)
    with pytest.raises(ValueError):
        mfcc_amd.running_norm_state(sums, -1.0)


@pytest.mark.parametrize("call", [
    # more threads than one launch counts (2^32 - 1): workgroups are sequences x column blocks
    # (2^20 columns: 8192 blocks of 64 pairs; 100 rows take a workgroup of 512 threads to themselves: 1024 x 8192 x 512 = 2^32)
    lambda l: scan(l, n=1024, steps=100, ncol=1 << 20, y=rows(100 << 20, 1 << 20)),
    lambda l: norm(l, n=1 << 24, steps=600, ncol=64, x=rows(38400, 64), y=rows(38400, 64)),
    lambda l: drop(l, n=1 << 24, steps=300, ncol=8, x=rows(2400, 8), y=rows(2400, 8)),
    lambda l: step(l, n=1 << 24, ncol=256, x_ld=256, y_ld=256),
    # products that would pass 63 bits
    lambda l: scan(l, n=1 << 24, steps=1 << 30, ncol=1 << 20, y=rows(1 << 50, 1 << 20)),
    lambda l: drop(l, n=1 << 24, steps=1 << 30, ncol=1 << 20, y=rows(1 << 50, 1 << 20)),
    lambda l: l.mfcc_gated_scan_checkpoints(None, 1 << 24, 1 << 30, 1 << 20, 0),
    lambda l: l.mfcc_sequence_workspace(None, 1 << 24, 1 << 30, 1 << 20, 0)])
def test_what_one_launch_does_not_cover_is_refused(lib, call):
    assert call(lib) == capi.ERR_UNSUPPORTED
    assert lib.mfcc_last_error()
