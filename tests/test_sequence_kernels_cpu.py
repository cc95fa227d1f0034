"""The kernels of the operators along time, built for the host from their own sources (tests/host_sim/sequence_sim.cpp): every
workgroup's LDS starts as NaN and its threads take turns at the barriers, so that a value used without having been written shows
on every run.  Compared with the definitions, row by row in 64 bits."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

capi = pytest.importorskip("mfcc_amd._capi")
HERE = os.path.dirname(os.path.abspath(__file__))
U = 2.0 ** -24   # half a step of float32


@pytest.fixture(scope="module")
def sim():
    subprocess.check_call(["make", "-C", os.path.dirname(HERE), "host_sim"])
    lib = C.CDLL(os.path.join(HERE, "host_sim", "libsequence_sim.so"))
    for name, (res, args) in capi.SIGNATURES.items():
        if hasattr(lib, name):
            f = getattr(lib, name)
            f.restype, f.argtypes = res, args
    lib.sim_layout.restype, lib.sim_layout.argtypes = C.c_void_p, [C.c_void_p, C.c_int64]
    lib.sim_layout_free.restype, lib.sim_layout_free.argtypes = None, [C.c_void_p]
    lib.sim_division.restype, lib.sim_division.argtypes = None, [C.c_int64, C.c_int64, C.c_int32, C.c_void_p]
    return lib


def division(sim, n, longest, d):
    """(columns of a group, groups of a block, groups of the last block, pieces)"""
    out = np.zeros(4, np.int32)
    sim.sim_division(n, longest, d, out.ctypes.data)
    return out.tolist()


def rows(a):
    return capi.MfccRows(a.ctypes.data, 0, a.shape[-1])


def ptr(a):
    return None if a is None else a.ctypes.data


class Layout:
    def __init__(self, sim, counts):
        self.sim, self.counts = sim, np.asarray(counts, np.int64)

    def __enter__(self):
        self.h = self.sim.sim_layout(self.counts.ctypes.data, len(self.counts))
        return self.h

    def __exit__(self, *_):
        self.sim.sim_layout_free(self.h)


def workspace(sim, lay, d):
    n = sim.mfcc_sequence_workspace(lay, 0, 0, d, capi.ROWS_F32)
    assert n >= 0
    raw = np.full(n // 4 + 8, np.nan, np.float32)
    return raw[(-raw.ctypes.data % 16) // 4:]


def norm_definition(x, decay, state, eps):
    d = x.shape[1]
    w, m, s = state[0], state[1:1 + d].copy(), state[1 + d:].copy()
    y, sig = np.zeros_like(x), np.zeros_like(x)
    for t in range(len(x)):
        w = decay * w + 1
        off = x[t] - m
        m = m + off / w
        s = decay * s + off * (x[t] - m)
        sig[t] = np.sqrt(s / w + eps)
        y[t] = (x[t] - m) / sig[t]
    return y, np.concatenate([[w], m, s]), sig


def check_norm(sim, counts, d, decay=0.97, seed=0, in_place=False, eps=1e-5):
    rng = np.random.default_rng(seed)
    n = len(counts)
    level, spread = rng.standard_normal(d) * 6, 0.5 + 3 * rng.random(d)
    x = (rng.standard_normal((sum(counts), d)) * spread + level).astype(np.float32)
    w = 5 + 100 * rng.random((n, 1))   # every sequence its own weight: another one's reciprocals are wrong here
    state = np.concatenate([w, level + rng.standard_normal((n, d)), w * spread ** 2], 1).astype(np.float32)
    src = x.copy()
    y = src if in_place else np.full_like(x, np.nan)
    end = np.full_like(state, np.nan)
    with Layout(sim, counts) as lay:
        ws = workspace(sim, lay, d)
        assert sim.mfcc_running_norm(lay, 0, 0, d, decay, eps, 0, rows(src), ptr(state), rows(y), 0, ptr(end), ptr(ws), None) == 0
    at = 0
    for u, c in enumerate(counts):
        xs, start = x[at:at + c].astype(np.float64), state[u].astype(np.float64)
        ref, fin, sig = norm_definition(xs, decay, start, eps)
        # as on the device: a few roundings of the size of the values in the mean, the deviation divides them by sigma, whose own relative
        # error is of the same size
        big = max(np.abs(xs).max(initial=0), np.abs(start[1:1 + d]).max())
        tol = 32 * U * (big / sig + np.abs(ref) * (1 + big / sig)) + U * np.abs(ref)
        bad = ~(np.abs(y[at:at + c] - ref) <= tol)
        assert not bad.any(), f"{bad.sum()} of {bad.size} off, columns {np.unique(np.nonzero(bad)[1])}"
        assert abs(end[u, 0] - fin[0]) <= 64 * U * fin[0]
        assert (np.abs(end[u, 1:1 + d] - fin[1:1 + d]) <= 32 * U * big).all()
        q = fin[1 + d:]
        assert (np.abs(end[u, 1 + d:] - q) <= 64 * U * (q + np.sqrt(q * max(fin[0], 1)) * big)).all()
        at += c


# widths whose last block of columns has 1 to 7 groups, and some that do not: (counts, columns, groups of the last block)
LAST_BLOCKS = [([100], 1285, 5), ([40, 3], 993, 1), ([70], 807, 7), ([70], 869, 5), ([60, 9], 1799, 7), ([70], 1025, 1), ([70] * 7, 1025, 1),
               ([50, 8], 2050, 1), ([70], 995, 3), ([8] * 64, 3655, 7), ([700], 4097, 1), ([33, 0, 5], 39, 39), ([90], 257, 25), ([40], 4369, 17)]


@pytest.mark.parametrize("counts,d,last", LAST_BLOCKS)
def test_norm_last_column_block(sim, counts, d, last):
    div = division(sim, len(counts), max(counts), d)
    assert div[2] == last and (div[3] > 1) == (counts == [700]), div
    check_norm(sim, counts, d, seed=d, in_place=bool(d % 4 == 1))
