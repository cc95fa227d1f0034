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


def workspace(sim, lay, d, steps=0):
    n = sim.mfcc_sequence_workspace(lay, 1, steps, d, capi.ROWS_F32)
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


# --------------------------------------------------------------------------
# the recurrence over sequences that are cut into pieces
# --------------------------------------------------------------------------
def run_scan(sim, x, g, h0=None, form=0, gy=None, glast=None):
    """One packed float32 sequence: (y, last[, dx, dg, dh0])"""
    n, d = x.shape
    none = C.c_void_p(None)
    head = none, 1, n, d, 0, form, 0
    y, last = np.full_like(x, np.nan), np.full(d, np.nan, np.float32)
    ws = workspace(sim, None, d, n)
    ck = np.full(sim.mfcc_gated_scan_checkpoints(None, 1, n, d, 0), np.nan, np.float32)
    assert sim.mfcc_gated_scan(*head, rows(x), rows(g), ptr(h0), rows(y), ptr(last), ptr(ck), ptr(ws), None) == 0
    if gy is None:
        return y, last
    dx, dg, dh = np.full_like(x, np.nan), np.full_like(x, np.nan), np.full(d, np.nan, np.float32)
    assert sim.mfcc_gated_scan_backward(*head, rows(x), rows(g), ptr(ck), rows(gy), ptr(glast), rows(dx), rows(dg), ptr(dh), ptr(ws), None) == 0
    return y, last, dx, dg, dh


def scan_definition(x, g, h0, form):
    a = g if form == 0 else 1 / (1 + np.exp(-g))
    b = x if form == 0 else x / (1 + np.exp(g))
    h, m = h0.copy(), np.abs(h0)
    y, mag, before = np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)
    for t in range(len(x)):
        before[t] = h
        h = a[t] * h + b[t]
        m = np.abs(a[t]) * m + np.abs(b[t])
        y[t], mag[t] = h, m
    return y, mag, a, before


def agree(got, ref, mag, length):
    """Equal where not finite, otherwise within 16 u for each of `length` rows and for their products"""
    fin = np.isfinite(ref)
    assert np.array_equal(got[~fin], ref[~fin], equal_nan=True)
    assert (np.abs(got[fin] - ref[fin]) <= 16 * U * (1 + length) * mag[fin] + 2.0 ** -149).all()


@pytest.mark.parametrize("form", [0, 1])
def test_infinite_states_stay_infinite(sim, form):
    """An infinity is carried over pieces whose products of gates vanish in 32 bits, forwards and backwards."""
    n, d = 6000, 8
    assert division(sim, 1, n, d)[3] > 1
    rng = np.random.default_rng(form)
    x, g, gy = (rng.standard_normal((n, d)).astype(np.float32) for _ in range(3))
    if form == 0:
        g = (1 / (1 + np.exp(-g))).astype(np.float32) * np.where(rng.random((n, d)) < 0.2, np.float32(-1), np.float32(1))
    x[100, 1], x[2000, 2], x[5500, 3] = np.inf, -np.inf, np.inf
    gy[5900, 4], gy[3000, 5] = np.inf, -np.inf
    h0, gl = rng.standard_normal(d).astype(np.float32), rng.standard_normal(d).astype(np.float32)
    h0[0], gl[6] = -np.inf, np.inf
    y, last, dx, dg, dh = run_scan(sim, x, g, h0, form, gy, gl)
    ref, mag, a, before = scan_definition(x.astype(np.float64), g.astype(np.float64), h0.astype(np.float64), form)
    # gates of at most 1 / (1 + exp(-5)): a memory below 150 rows
    agree(y, ref, mag, 150)
    agree(last, ref[-1], mag[-1], 150)
    assert np.isinf(ref[-1]).sum() == 4
    e, em, finite = gl.astype(np.float64), np.abs(gl).astype(np.float64), np.isfinite(before) & np.isfinite(x)
    na = np.ones_like(a) if form == 0 else 1 / (1 + np.exp(g.astype(np.float64)))
    ex, exm, eg, egm = (np.zeros_like(ref) for _ in range(4))
    for t in reversed(range(n)):
        delta, dm = gy[t] + e, np.abs(gy[t]) + em
        ex[t], exm[t] = na[t] * delta, na[t] * dm
        with np.errstate(invalid="ignore"):
            eg[t] = delta * before[t] if form == 0 else delta * a[t] * na[t] * (before[t] - x[t])
            egm[t] = dm * np.maximum(mag[t - 1] if t else np.abs(h0), np.abs(x[t]))
        e, em = a[t] * delta, np.abs(a[t]) * dm
    agree(dx, ex, exm, 150)
    agree(dh, e, em, 150)
    agree(dg[finite], eg[finite], 2 * egm[finite], 300)


def test_products_of_gates_past_32_bits(sim):
    """Gates above 1 whose product overflows while the states stay finite: nothing there to grow, or a gate of 0 afterwards."""
    n, d = 6000, 8
    assert division(sim, 1, n, d)[3] > 1
    rng = np.random.default_rng(3)
    x = rng.standard_normal((n, d)).astype(np.float32)
    g = np.full((n, d), 0.9, np.float32)
    g[:4000, :4] = 1.1           # 1.1 ** 1536, a piece: 4e63
    x[:3900, 0] = 0              # rows of 0 until shortly before they end
    x[:4000, 1], g[4000, 1] = 0, 0
    g[:4001:500, 2] = 0          # 1.1 ** 500 = 5e20 in between
    g[:4000, 3], x[:4000, 3] = -1.1, 0
    h0 = np.zeros(d, np.float32)
    h0[4:] = 1e30
    y, last = run_scan(sim, x, g, h0)
    ref, mag, _, _ = scan_definition(x.astype(np.float64), g.astype(np.float64), h0.astype(np.float64), 0)
    assert np.isfinite(ref).all() and np.abs(ref).max() < 3e38
    agree(y, ref, mag, n)
    agree(last, ref[-1], mag[-1], n)


# --------------------------------------------------------------------------
# values at the ends of the range of the normalisation
# --------------------------------------------------------------------------
def small_variances(rng, n, d):
    """Rows around 0 whose variances lie from 2^-140 to 2^-120, where the smallest normal number is 2^-126"""
    return (rng.standard_normal((n, d)) * 2.0 ** rng.uniform(-70, -60, d)).astype(np.float32)


def small_variance_tolerance(x, ref, decay, fin):
    """A subnormal sum of squares is off by half a step, 2^-150, for each of its two roundings a row, all of which decay like the rows:
    2^-149 / (1 - decay) in all, relative to the sum s halved by the root; the 32 u of the other roundings on top."""
    s = np.zeros(x.shape[1])
    rel = np.zeros_like(x)
    m, w = np.zeros(x.shape[1]), 0.0
    for t in range(len(x)):
        w = decay * w + 1
        off = x[t] - m
        m = m + off / w
        s = decay * s + off * (x[t] - m)
        rel[t] = 2.0 ** -149 / (1 - decay) / np.maximum(s, 1e-300)
    return np.abs(ref) * (rel + 64 * U), rel < 0.1


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -149, 2.0 ** -127])
def test_norm_of_subnormal_variances(sim, eps):
    rng, n, d, decay = np.random.default_rng(5), 300, 24, 0.9
    x = small_variances(rng, n, d)
    y = np.full_like(x, np.nan)
    assert sim.mfcc_running_norm(None, 1, n, d, decay, eps, 0, rows(x), None, rows(y), 0, None, None, None) == 0
    with np.errstate(invalid="ignore"):
        ref, fin, _ = norm_definition(x.astype(np.float64), decay, np.zeros(1 + 2 * d), eps)
    tol, known = small_variance_tolerance(x.astype(np.float64), ref, decay, fin)
    known[0] = False             # 0 / sqrt(eps) of the first row
    assert known.mean() > 0.5 and (np.abs(y - ref)[known] <= tol[known] + 32 * U * 8).all()   # means of values below 8 sigma


@pytest.mark.parametrize("w0", [0.0, 2.0 ** -30, 2.0 ** -10])
def test_norm_from_a_state_without_weight(sim, w0):
    """Means far away that carry no weight leave nothing behind."""
    rng, d = np.random.default_rng(6), 40
    for n in (1, 5, 40, 3000):
        x = (rng.standard_normal((n, d)) * 3 + 7).astype(np.float32)
        st = np.concatenate([[w0], rng.standard_normal(d) * 1000, np.zeros(d)]).astype(np.float32)
        y, end = np.full_like(x, np.nan), np.full_like(st, np.nan)
        ws = workspace(sim, None, d, n)
        assert sim.mfcc_running_norm(None, 1, n, d, 0.9, 1e-5, 0, rows(x), ptr(st), rows(y), 0, ptr(end), ptr(ws), None) == 0
        counted = st.astype(np.float64) if w0 > 2.0 ** -22 else np.zeros(1 + 2 * d)
        ref, fin, sig = norm_definition(x.astype(np.float64), 0.9, counted, 1e-5)
        big = max(np.abs(x).max(), np.abs(counted[1:1 + d]).max())
        assert (np.abs(y - ref) <= 32 * U * (big / sig + np.abs(ref) * (1 + big / sig)) + U * np.abs(ref)).all()
        assert (np.abs(end[1:1 + d] - fin[1:1 + d]) <= 32 * U * big).all()
        if w0 < 2.0 ** -22:
            assert not y[0].any()
