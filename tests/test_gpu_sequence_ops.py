"""The operators along time (mfcc_amd.recurrent) against their definitions, frame by frame in 64 bits
on the host.

Tolerances.  u = 2^-24 is half a step of float32, e_T half a step of the rows' type T (2^-24, 2^-8, 2^-11 of a
value for float32, bfloat16, float16: torch.finfo(T).eps / 2).  A state of the recurrence is a
sum of terms; each of its steps rounds once or twice, and every rounding decays with the gates that
follow it, so its error is at most a few u times M = sum of the absolute terms (the same recurrence over absolute values): per
step one product-sum (1 u), the gate's exponential, sum, reciprocal and product (8 u in all: |g| <= 8 costs |g| log2(e) / 2
steps in the exponent, the rest one step each), and the compositions that carry a state over a tile (1 u for every row of the product of gates, a
decaying sum, counted again).  An error made at one row reaches every later one with the weight of its term, so a memory of
L rows sees at most L of them: tolerance 16 u (1 + L) M with L <= min(rows, 1 / (1 - largest gate)), plus e_T |y|."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # steps of the subnormals


@pytest.fixture(scope="module")
def M():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    import mfcc_amd
    return mfcc_amd


def host(t):
    return t.detach().double().cpu().numpy()


def cell(x, g, form):
    """(a, 1 - a or 1, additive term) of one frame"""
    if form == "decay":
        return g, np.ones_like(g), x
    a, na = 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))
    return a, na, na * x


def sequence(x, g, h0, form, reverse, gy=None, glast=None):
    """One sequence [n, D] in 64 bits, and beside every result its magnitude (the same sums over absolute values):
    (y, last[, dx, dg, dh0]) and (|y|, ...)"""
    order = slice(None, None, -1) if reverse else slice(None)
    x, g = x[order], g[order]
    n = len(x)
    h, hm = h0.copy(), np.abs(h0)
    y, ym, before, beforem = (np.zeros_like(x) for _ in range(4))
    for t in range(n):
        a, na, b = cell(x[t], g[t], form)
        before[t], beforem[t] = h, hm
        h = a * h + b
        hm = np.abs(a) * hm + np.abs(b)
        y[t], ym[t] = h, hm
    out, mag = [y[order], h], [ym[order], hm]
    if gy is not None:
        gy = gy[order]
        e, em = glast.copy(), np.abs(glast)
        dx, dxm, dg, dgm = (np.zeros_like(x) for _ in range(4))
        for t in reversed(range(n)):
            a, na, _ = cell(x[t], g[t], form)
            d, dm = gy[t] + e, np.abs(gy[t]) + em
            dx[t], dxm[t] = na * d, na * dm
            k = 1.0 if form == "decay" else a * na
            off = 0.0 if form == "decay" else x[t]
            dg[t], dgm[t] = k * d * (before[t] - off), k * dm * (beforem[t] + np.abs(off))
            e, em = a * d, np.abs(a) * dm
        out += [dx[order], dg[order], e]
        mag += [dxm[order], dgm[order], em]
    return out, mag


def memory(g, form, n):
    if g.size == 0:
        return 1
    a = np.abs(g if form == "decay" else 1 / (1 + np.exp(-g))).max()
    return min(n, 1 / max(1e-9, 1 - a))


def close(got, ref, mag, dtype, mem, what):
    got = host(got)
    tol = 16 * U * (1 + mem) * mag + HALF[dtype] * np.abs(ref) + TINY[dtype]
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.abs(got - ref)[bad].max()} against {tol[bad].min()}"


def make_gate(gen, shape, form, dtype):
    g = torch.randn(shape, generator=gen, device="cuda") * 1.5 + 2
    g = g.clamp(-8, 8)
    if form == "decay":
        g = torch.sigmoid(g) * torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.1, -1.0, 1.0)
        g = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.05, 0.0, g)   # a gate of 0 starts afresh
    return g.to(dtype)


COUNTS = {"one": [1], "few": [7, 0, 1, 9, 8, 64, 3], "long": [2111], "mixed": [300, 1, 0, 97, 700, 16], "empty": [0, 0], "many": [5] * 300,
          "ends": [511, 512, 513, 104, 105]}


def check_scan(M, counts, d, dtype, form, reverse=False, padded=None, h0=True, train=True, seed=0, strided=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = len(counts)
    shape = (n, padded, d) if padded is not None else (sum(counts), d)
    x, g, gy = (torch.randn(shape, generator=gen, device="cuda").to(dtype) for _ in range(3))
    g = make_gate(gen, shape, form, dtype)
    if strided:   # views into larger tensors at odd offsets
        def view(t):
            wide = torch.full((*t.shape[:-1], d + 5), float("nan"), dtype=dtype, device="cuda")
            wide[..., 3:3 + d] = t
            return wide[..., 3:3 + d]
        x, g, gy = view(x), view(g), view(gy)
    h = torch.randn(n, d, generator=gen, device="cuda") if h0 else None
    glast = torch.randn(n, d, generator=gen, device="cuda")
    leaves = [t for t in (x, g, h) if t is not None]
    if train:
        for t in leaves:
            t.requires_grad_(True)
    y, last = M.gated_scan(x, g, counts, h0=h, form=form, reverse=reverse)
    assert y.shape == x.shape and y.dtype == dtype and last.shape == (n, d) and last.dtype == torch.float32
    grads = torch.autograd.grad((y, last), leaves, (gy, glast)) if train else ()
    if not train:
        y2, last2 = M.gated_scan(x, g, counts, h0=h, form=form, reverse=reverse)
        assert torch.equal(y, y2) and torch.equal(last, last2)
    xs, gs, gys, ys = host(x), host(g), host(gy), y.detach()
    at = 0
    for u, c in enumerate(counts):
        c = c if padded is None else min(c, padded)
        sl = (u, slice(0, c)) if padded is not None else (slice(at, at + c),)
        at += c
        start = host(h)[u] if h0 else np.zeros(d)
        out, mag = sequence(xs[sl], gs[sl], start, form, reverse, gys[sl] if train else None, host(glast)[u])
        mem = memory(gs[sl], form, c)
        where = f"sequence {u} of {c}"
        close(ys[sl], out[0], mag[0], dtype, mem, "y " + where)
        close(last[u], out[1], mag[1], torch.float32, mem, "last " + where)
        if c == 0:
            assert np.array_equal(host(last[u]), start)
        if train:
            # the gradients hold a product of two such sums
            close(grads[0][sl], out[2], mag[2], dtype, mem, "dx " + where)
            close(grads[1][sl], out[3], mag[3], dtype, 2 * mem, "dgate " + where)
            if h0:
                close(grads[2][u], out[4], mag[4], torch.float32, mem, "dh0 " + where)
        if padded is not None:
            for t in (ys,) + tuple(grads[:2]):
                assert not t[u, c:].any(), "rows behind the end of a padded sequence hold 0"
    return y, last, grads


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("d", [1, 39, 64])
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
def test_scan_lengths(M, name, d, form):
    check_scan(M, COUNTS[name], d, torch.float32, form, seed=len(name) + d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [2, 3, 8, 40, 130, 257, 516])
def test_scan_columns_and_types(M, dtype, d):
    for form, reverse in (("decay", True), ("sigmoid", False)):
        check_scan(M, [33, 0, 140, 1], d, dtype, form, reverse=reverse, seed=d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_padded(M, dtype, reverse):
    for d in (39, 64):
        check_scan(M, [50, 0, 70, 1, 90], d, dtype, "sigmoid", reverse=reverse, padded=70, seed=d)    # 90 counts as 70
    check_scan(M, [3, 3], 5, dtype, "decay", reverse=reverse, padded=3, h0=False)


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.float16, 39)])
def test_scan_views(M, dtype, d):
    """Odd element offsets and row strides, surrounded by NaN."""
    check_scan(M, [130, 5], d, dtype, "sigmoid", strided=True, seed=1)
    check_scan(M, [40, 61], d, dtype, "decay", strided=True, padded=61, reverse=True, seed=2)


@pytest.mark.parametrize("d,rows,n", [(39, 20000, 1), (64, 9000, 2), (257, 5000, 1)])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_long(M, d, rows, n, reverse):
    """Few long sequences: the time axis is split over workgroups and joined."""
    counts = [rows - 77 * k for k in range(n)]
    check_scan(M, counts, d, torch.float32, "sigmoid", reverse=reverse, seed=3)
    check_scan(M, counts, d, torch.bfloat16, "decay", reverse=reverse, seed=4, h0=False)
    check_scan(M, counts, d, torch.float16, "sigmoid", reverse=reverse, seed=5, padded=rows + 9, train=False)


def test_scan_pieces_equal_the_whole(M):
    """last of one piece is h0 of the next; the step form walks the same states."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, g = torch.randn(4, 60, 48, generator=gen, device="cuda"), torch.randn(4, 60, 48, generator=gen, device="cuda")
    y, last = M.gated_scan(x, g, form="sigmoid")
    a, mid = M.gated_scan(x[:, :23], g[:, :23], form="sigmoid")
    b, end = M.gated_scan(x[:, 23:], g[:, 23:], h0=mid, form="sigmoid")
    # two paths of the same sums: 16 u (1 + 23) of magnitudes below 8 as in the comparison with 64 bits, twice
    tol = 2 * 16 * U * 24 * 8
    assert (torch.cat([a, b], 1) - y).abs().max() <= tol and (end - last).abs().max() <= tol
    state = torch.zeros(4, 48, device="cuda")
    for t in range(60):
        row, state = M.gated_scan_step(x[:, t], g[:, t], state, form="sigmoid", state_out=state if t % 2 else None)
        assert torch.equal(row, state) and (row - y[:, t]).abs().max() <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d", [(1, 1), (64, 512), (3, 39), (7, 1030)])
def test_step(M, dtype, n, d):
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    x, h = torch.randn(n, d, generator=gen, device="cuda").to(dtype), torch.randn(n, d, generator=gen, device="cuda")
    for form in ("decay", "sigmoid"):
        g = make_gate(gen, (n, d), form, dtype)
        y, s = M.gated_scan_step(x, g, h, form=form)
        a, na, b = cell(host(x), host(g), form)
        ref = a * host(h) + b
        mag = np.abs(a * host(h)) + np.abs(b)
        close(y, ref, mag, dtype, 1, "y")
        close(s, ref, mag, torch.float32, 1, "state")
        wide = torch.full((n, d + 3), float("nan"), dtype=dtype, device="cuda")
        out = torch.full((n, d + 7), -7.0, dtype=dtype, device="cuda")
        wide[:, 1:1 + d] = x
        h2 = h.clone()
        y2, s2 = M.gated_scan_step(wide[:, 1:1 + d], g, h2, form=form, out=out[:, 2:2 + d], state_out=h2)
        assert torch.equal(y2, y) and torch.equal(s2, s) and s2 is h2
        assert (out[:, :2] == -7).all() and (out[:, 2 + d:] == -7).all()


def test_scan_gradient_against_differences(M):
    gen = torch.Generator(device="cuda").manual_seed(8)
    counts, d = [9, 1, 21], 3
    for form in ("decay", "sigmoid"):
        x, g = torch.randn(31, d, generator=gen, device="cuda"), make_gate(gen, (31, d), form, torch.float32)
        h0, wy, wl = torch.randn(3, d, generator=gen, device="cuda"), torch.randn(31, d, generator=gen, device="cuda"), torch.randn(3, d, generator=gen, device="cuda")
        leaves = [t.clone().requires_grad_(True) for t in (x, g, h0)]
        y, last = M.gated_scan(leaves[0], leaves[1], counts, h0=leaves[2], form=form)
        grads = torch.autograd.grad((y * wy).sum() + (last * wl).sum(), leaves)

        def loss(vals):
            y, last = M.gated_scan(vals[0], vals[1], counts, h0=vals[2], form=form)
            return float((y.double() * wy.double()).sum() + (last.double() * wl.double()).sum())

        for k in range(3):
            direction = torch.randn(leaves[k].shape, generator=gen, device="cuda")
            step = 1e-2
            up, down = ([t.detach() + (s * step * direction if i == k else 0) for i, t in enumerate(leaves)] for s in (1, -1))
            slope = (loss(up) - loss(down)) / (2 * step)
            want = float((grads[k].double() * direction.double()).sum())
            # central differences: third derivatives over 1e-4 / 6 of sums of a few hundred terms of size 1, and 2^-24 of those sums over 1e-2
            assert abs(slope - want) <= 2e-2 * (1 + abs(want)), (form, k, slope, want)


def test_scan_partial_gradients_and_broadcast_gate(M):
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(50, 12, generator=gen, device="cuda")
    lam = torch.rand(12, generator=gen, device="cuda").requires_grad_(True)
    y, last = M.gated_scan(x, lam.expand(50, 12), [20, 30])
    (dl,) = torch.autograd.grad(last.sum(), lam)        # no gradient arrives at y
    full = lam.detach().expand(50, 12).clone().requires_grad_(True)
    y2, last2 = M.gated_scan(x, full, [20, 30])
    (df,) = torch.autograd.grad(last2.sum(), full)
    assert torch.equal(y, y2)
    assert torch.allclose(dl, df.sum(0), rtol=0, atol=50 * U * float(df.abs().sum(0).max()))
    xr = x.clone().requires_grad_(True)
    y3, _ = M.gated_scan(xr, full.detach(), [20, 30])
    (dx,) = torch.autograd.grad(y3.sum(), xr)            # only x, only through y, a gradient of expanded ones
    ref = torch.cat([torch.from_numpy(sequence(host(x)[s], host(full)[s], np.zeros(12), "decay", False, np.ones((n, 12)), np.zeros(12))[0][2])
                     for s, n in ((slice(0, 20), 20), (slice(20, 50), 30))])
    assert (dx.cpu().double() - ref).abs().max() <= 16 * U * 31 * float(ref.abs().max())


def test_scan_nonfinite_stay_inside_their_sequence_and_column(M):
    x = torch.randn(3, 40, 70, device="cuda")
    g = torch.randn(3, 40, 70, device="cuda")
    clean, _ = M.gated_scan(x, g, form="sigmoid")
    x[1, 11, 33] = float("nan")
    x[1, 20, 5] = float("inf")
    y, _ = M.gated_scan(x, g, form="sigmoid")
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[1, 11:, 33] = True
    touched[1, 20:, 5] = True
    assert torch.equal(y[~touched], clean[~touched])
    assert torch.isnan(y[1, 11:, 33]).all() and not torch.isfinite(y[1, 20:, 5]).any()
    # extreme gates: a = 1 and a = 0 exactly
    g2 = torch.full((1, 30, 4), 200.0, device="cuda")
    g2[0, 15:] = -200.0
    x2 = torch.randn(1, 30, 4, device="cuda")
    h0 = torch.randn(1, 4, device="cuda")
    y2, _ = M.gated_scan(x2, g2, h0=h0, form="sigmoid")
    assert torch.equal(y2[0, :15], h0.expand(15, 4)) and torch.equal(y2[0, 15:], x2[0, 15:])


def test_scan_out_and_in_place(M):
    x, g = torch.randn(90, 39, device="cuda"), torch.rand(90, 39, device="cuda")
    y, last = M.gated_scan(x, g, [40, 50])
    buf = torch.full((92, 48), 5.0, device="cuda")
    y2, last2 = M.gated_scan(x, g, [40, 50], out=buf[1:91, 4:43])
    assert torch.equal(y2, y) and torch.equal(last, last2)
    assert (buf[0] == 5).all() and (buf[91] == 5).all() and (buf[:, :4] == 5).all() and (buf[:, 43:] == 5).all()
    same, _ = M.gated_scan(x, g, [40, 50], out=x)
    assert same is x and torch.equal(x, y)
    tm = torch.empty(30, 4, 8, device="cuda").transpose(0, 1)      # time-major memory
    x3, g3 = torch.randn(4, 30, 8, device="cuda"), torch.rand(4, 30, 8, device="cuda")
    assert torch.equal(M.gated_scan(x3, g3, out=tm)[0], M.gated_scan(x3, g3)[0])


# --------------------------------------------------------------------------
# running normalisation
# --------------------------------------------------------------------------
def norm_sequence(x, lam, state, eps, center_only):
    d = x.shape[1]
    w, m, s = state[0], state[1:1 + d].copy(), state[1 + d:].copy()
    y = np.zeros_like(x)
    for t in range(len(x)):
        w = lam * w + 1
        off = x[t] - m
        m = m + off / w
        s = lam * s + off * (x[t] - m)
        y[t] = (x[t] - m) if center_only else (x[t] - m) / np.sqrt(s / w + eps)
    return y, np.concatenate([[w], m, s])


def check_norm(M, counts, d, decay, dtype=torch.float32, state=True, padded=None, center_only=False, seed=0, eps=1e-5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = len(counts)
    shape = (n, padded, d) if padded is not None else (sum(counts), d)
    level, spread = torch.randn(d, generator=gen, device="cuda") * 6, 0.5 + 3 * torch.rand(d, generator=gen, device="cuda")
    x = torch.randn(shape, generator=gen, device="cuda") * spread + level
    st = None
    if state:
        w = 5 + 100 * torch.rand(n, 1, generator=gen, device="cuda")
        st = torch.cat([w, level + torch.randn(n, d, generator=gen, device="cuda"), w * spread ** 2], 1)
    y, end = M.running_norm(x, counts, decay=decay, state=st, center_only=center_only, dtype=dtype, eps=eps)
    assert y.dtype == dtype and y.shape == x.shape and end.shape == (n, 1 + 2 * d)
    at, lam = 0, decay
    for u, c in enumerate(counts):
        c = c if padded is None else min(c, padded)
        sl = (u, slice(0, c)) if padded is not None else (slice(at, at + c),)
        at += c
        start = host(st)[u] if state else np.zeros(1 + 2 * d)
        xs = host(x)[sl]
        ref, fin = norm_sequence(xs, lam, start, eps, center_only)
        # a mean of values of size |x| <= X moves by u X at every rounding (about four a row: difference, product, sum,
        # reciprocal), and a row's rounding decays like its weight: at most min(rows, 1 / (1 - decay)) of them of
        # weight 1 / w each, so a few u X in all for the mean; the composition of the runs that a tile joins adds as many.
        # 32 u X for x - m; the deviation divides it by sigma = sqrt(s / w + eps), whose own relative error is
        # 32 u (1 + X / sigma) again, on a quotient that is at most |y|
        big = max(np.abs(xs).max(initial=0), np.abs(start[1:1 + d]).max(initial=0))
        off = ref if center_only else None
        if center_only:
            tol = 32 * U * big + HALF[dtype] * np.abs(ref) + TINY[dtype]
        else:
            sig = np.zeros_like(ref)
            w, m, s = start[0], start[1:1 + d].copy(), start[1 + d:].copy()
            for t in range(c):
                w = lam * w + 1
                dv = xs[t] - m
                m = m + dv / w
                s = lam * s + dv * (xs[t] - m)
                sig[t] = np.sqrt(s / w + eps)
            tol = 32 * U * (big / sig + np.abs(ref) * (1 + big / sig)) + HALF[dtype] * np.abs(ref) + TINY[dtype]
        got = host(y[sl])
        bad = ~(np.abs(got - ref) <= tol)
        assert not bad.any(), f"sequence {u} of {c}: {bad.sum()} off, worst {np.abs(got - ref)[bad].max()} against {tol[bad].min()}"
        e = host(end)[u]
        assert abs(e[0] - fin[0]) <= 64 * U * fin[0]
        assert (np.abs(e[1:1 + d] - fin[1:1 + d]) <= 32 * U * big).all()
        q = fin[1 + d:]
        assert (np.abs(e[1 + d:] - q) <= 64 * U * (q + np.sqrt(q * max(fin[0], 1)) * big)).all()
        if padded is not None:
            assert not y[u, c:].any()
    return x, y, end


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("d", [1, 13, 39, 64, 257])
def test_norm_lengths(M, name, d):
    check_norm(M, COUNTS[name], d, 0.99, state=bool(d % 2), seed=d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("decay", [0.5, 0.95, 0.9995, 1.0])
def test_norm_decays_and_types(M, dtype, decay):
    check_norm(M, [33, 0, 700, 1], 40, decay, dtype=dtype, seed=1)
    check_norm(M, [20, 50, 60], 39, decay, dtype=dtype, state=False, padded=50, seed=2)
    check_norm(M, [20, 50], 39, decay, dtype=dtype, center_only=True, seed=3)


@pytest.mark.parametrize("decay", [0.995, 1.0])
def test_norm_long(M, decay):
    for d, rows in ((39, 20000), (64, 9001), (257, 4000)):
        check_norm(M, [rows], d, decay, seed=d)
        check_norm(M, [rows, 5, rows // 2], d, decay, state=False, padded=rows + 3, dtype=torch.bfloat16, seed=d)


def test_norm_constant_columns_and_first_rows(M):
    x = torch.full((2, 50, 7), 17.3, device="cuda")
    y, end = M.running_norm(x, decay=0.9)
    assert not y.any() and torch.equal(end[:, 1:8], x[:, 0]) and not end[:, 8:].any()
    x = torch.randn(5, 1, 9, device="cuda") * 50
    assert not M.running_norm(x)[0].any()     # a first row is its own mean


def test_norm_pieces_equal_the_whole_and_prior(M):
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(3, 200, 39, generator=gen, device="cuda") * 4 + 2
    sums = M.cmvn_accumulate(x.reshape(-1, 39))
    prior = M.running_norm_state(sums, 50.0, n_seq=3)
    assert torch.equal(prior[:, 0], torch.full((3,), 50.0, device="cuda"))
    y, end = M.running_norm(x, decay=0.98, state=prior)
    state, parts = prior, []
    for a, b in ((0, 1), (1, 64), (64, 65), (65, 200)):
        p, state = M.running_norm(x[:, a:b], decay=0.98, state=state)
        parts.append(p)
    assert (torch.cat(parts, 1) - y).abs().max() <= 2 * 32 * U * 30 * 4        # both within the tolerance above of the same values
    assert (state - end).abs().max() <= 2 * 64 * U * 1e4
    xi = x.clone()
    yi, _ = M.running_norm(xi, decay=0.98, state=prior, out=xi)
    assert yi is xi and torch.equal(xi, y)


def test_norm_nonfinite_stay_in_their_column(M):
    x = torch.randn(2, 90, 39, device="cuda")
    clean, _ = M.running_norm(x)
    x[0, 30, 7] = float("nan")
    y, _ = M.running_norm(x)
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[0, 30:, 7] = True
    assert torch.equal(y[~touched], clean[~touched]) and torch.isnan(y[touched]).all()


# --------------------------------------------------------------------------
# dropout
# --------------------------------------------------------------------------
def fields(e, step, seed):
    """16-bit fields of the elements e (uint64), Philox4x32-10 in numpy."""
    word, c = np.uint64(0xFFFFFFFF), [None] * 4
    block = e >> np.uint64(3)
    c = [block & word, block >> np.uint64(32), np.full_like(e, step % 2**32), np.full_like(e, step >> 32)]
    for i in range(10):
        k0, k1 = np.uint64((seed + i * 0x9E3779B9) % 2**32), np.uint64(((seed >> 32) + i * 0xBB67AE85) % 2**32)
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ k0, b & word, (a >> np.uint64(32)) ^ c[3] ^ k1, a & word]
    k = (e & np.uint64(7)).astype(int)
    w = np.choose(k >> 1, c)
    return np.where(k & 1, w >> np.uint64(16), w & np.uint64(0xFFFF))


def keep_mask(shape, counts, per, p, seed, step):
    d = shape[-1]
    if len(shape) == 3:
        u, r = np.repeat(np.arange(shape[0]), shape[1]), np.arange(shape[0] * shape[1])
    else:
        u = np.repeat(np.arange(len(counts)), counts) if counts is not None else np.zeros(shape[0], int)
        r = np.arange(shape[0])
    u, r, c = u.astype(np.uint64)[:, None], r.astype(np.uint64)[:, None], np.arange(d, dtype=np.uint64)
    e = r * np.uint64(d) + c if per == "element" else r + 0 * c if per == "frame" else u * np.uint64(-(-d // 8) * 8) + c
    return (fields(e, step, seed) >= int(round(p * 65536))).reshape(shape)


def check_dropout(M, shape, counts, per, p, dtype, seed, step, view=False):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    if view:
        wide = torch.full((*shape[:-1], shape[-1] + 5), float("nan"), dtype=dtype, device="cuda")
        wide[..., 3:3 + shape[-1]] = x
        x = wide[..., 3:3 + shape[-1]]
    keep = keep_mask(shape, counts, per, p, seed, step)
    thr = int(round(p * 65536))
    scale = 65536 / (65536 - thr) if thr < 65536 else 0.0
    gy = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    y = M.feature_dropout(x.requires_grad_(True), p, seed, step=step, per=per, frame_counts=counts)
    (dx,) = torch.autograd.grad(y, x, gy)
    for got, src in ((y, x), (dx, gy)):
        ref = host(src) * scale * keep
        # the product with a scale rounded to 24 bits, then the type: u + u + e_T
        tol = (2 * U + HALF[dtype]) * np.abs(ref) + TINY[dtype]
        assert got.dtype == dtype and (np.abs(host(got) - ref) <= tol).all()
        assert np.array_equal(host(got) == 0, ~keep | (host(src) == 0))
    return keep


@pytest.mark.parametrize("per", ["element", "frame", "sequence"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dropout_masks(M, per, dtype):
    for d in (1, 7, 39, 64, 129):
        counts = [3, 0, 50, 1, 12]
        check_dropout(M, (66, d), counts, per, 0.3, dtype, 0x123456789ABCDEF0 + d, (1 << 40) + 17)
        check_dropout(M, (4, 9, d), None, per, 0.5, dtype, d, 0)
    check_dropout(M, (66, 40), [66], per, 0.25, dtype, 2 ** 64 - 1, 2 ** 63 - 1, view=True)
    check_dropout(M, (3, 5, 24), None, per, 0.25, dtype, 7, 3, view=True)


def test_dropout_statistics(M):
    keep = check_dropout(M, (3000, 257), None, "element", 0.2, torch.float32, 99, 5)
    n = keep.size
    # a fair stream: the share kept lies within 6 standard deviations, columns and rows do not follow each other
    assert abs(keep.mean() - 0.8) <= 6 * np.sqrt(0.16 / n)
    z = keep - keep.mean()
    for lag in (1, 2, 8, 257, 514):
        a = z.reshape(-1)
        assert abs((a[lag:] * a[:-lag]).mean()) <= 6 * 0.16 / np.sqrt(n)
    other = keep_mask((3000, 257), None, "element", 0.2, 99, 6)
    assert abs((z * (other - other.mean())).mean()) <= 6 * 0.16 / np.sqrt(n)


def test_dropout_edges(M):
    x = torch.randn(40, 39, device="cuda")
    assert torch.equal(M.feature_dropout(x, 0.0, 1), x)
    assert not M.feature_dropout(x, 1.0, 1).any()
    x[3, 5], x[4, 6] = float("nan"), float("inf")
    assert not M.feature_dropout(x, 1.0, 1).any()
    y = M.feature_dropout(x, 0.5, 11, per="frame")
    gone = ~torch.from_numpy(keep_mask((40, 39), None, "frame", 0.5, 11, 0)).cuda()
    assert not y[gone].any()
    z = x.clone()
    out = M.feature_dropout(z, 0.5, 11, out=z)
    assert out is z and torch.equal(z.isnan(), M.feature_dropout(x, 0.5, 11).isnan())
    assert M.feature_dropout(x[:0], 0.5, 1).shape == (0, 39)
    step = torch.tensor([41], device="cuda")
    w = torch.randn(40, 39, device="cuda")
    assert torch.equal(M.feature_dropout(w, 0.5, 1, step=step), M.feature_dropout(w, 0.5, 1, step=41))
    w.requires_grad_(True)
    y = M.feature_dropout(w, 0.5, 1, step=step)
    step += 1
    with pytest.raises(RuntimeError):       # the mask of the backward pass would be another one
        y.sum().backward()


# --------------------------------------------------------------------------
# refusals, streams, graphs, the paths that call them
# --------------------------------------------------------------------------
def test_refusals(M):
    x, g = torch.randn(10, 8, device="cuda"), torch.rand(10, 8, device="cuda")
    bad = [lambda: M.gated_scan(x.cpu(), g.cpu()), lambda: M.gated_scan(x.double(), g.double()), lambda: M.gated_scan(x, g.half()),
           lambda: M.gated_scan(x, g[:5]), lambda: M.gated_scan(x, g, [4, 5]), lambda: M.gated_scan(x, g, [11, -1]),
           lambda: M.gated_scan(x, g, form="tanh"), lambda: M.gated_scan(x.t(), g.t()), lambda: M.gated_scan(x, g[:, :1].expand(10, 8)),
           lambda: M.gated_scan(x, g, [10], h0=torch.zeros(2, 8, device="cuda")), lambda: M.gated_scan(x, g, h0=torch.zeros(1, 8, device="cuda").half()),
           lambda: M.gated_scan(x, g, out=torch.empty(10, 9, device="cuda")), lambda: M.gated_scan(x.requires_grad_(True), g, out=torch.empty_like(g)),
           lambda: M.gated_scan(x[None, None], g[None, None]), lambda: M.gated_scan(x[None], g[None], [3, 4]),
           lambda: M.gated_scan_step(x, g, torch.zeros(10, 8, device="cuda")),     # x requires a gradient by now
           lambda: M.gated_scan_step(g, g, torch.zeros(10, 7, device="cuda")), lambda: M.gated_scan_step(g, g, None),
           lambda: M.gated_scan_step(g, g, torch.zeros(8, 10, device="cuda").t()),
           lambda: M.running_norm(x), lambda: M.running_norm(g, decay=0.0), lambda: M.running_norm(g, decay=1.01), lambda: M.running_norm(g.half()),
           lambda: M.running_norm(g, dtype=torch.float64), lambda: M.running_norm(g, state=torch.zeros(1, 16, device="cuda")),
           lambda: M.feature_dropout(g, 1.5, 0), lambda: M.feature_dropout(g, float("nan"), 0), lambda: M.feature_dropout(g, 0.5, -1),
           lambda: M.feature_dropout(g, 0.5, 1 << 64), lambda: M.feature_dropout(g, 0.5, 0, step=-1), lambda: M.feature_dropout(g, 0.5, 0, per="row"),
           lambda: M.feature_dropout(g, 0.5, 0, step=torch.tensor([1])), lambda: M.feature_dropout(g, 0.5, 0, frame_counts=[3])]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError(f"call {k} was accepted")
    from mfcc_amd import _capi as capi
    overlap = torch.empty(100, device="cuda").as_strided((10, 8), (4, 1))
    with pytest.raises(capi.MfccError):
        M.gated_scan(g, g, out=overlap)
    st = torch.zeros(1, 17, device="cuda")
    with pytest.raises(ValueError):
        M.running_norm(g, state=st, state_out=st)
    with pytest.raises(capi.MfccError):
        M.running_norm(g, eps=-1.0)


def test_empty_batches(M):
    e = torch.empty(0, 5, device="cuda")
    y, last = M.gated_scan(e, e)
    assert y.shape == (0, 5) and not last.any()
    h0 = torch.randn(3, 5, device="cuda", requires_grad=True)
    y, last = M.gated_scan(e, e, [0, 0, 0], h0=h0)
    (dh,) = torch.autograd.grad(last, h0, torch.ones(3, 5, device="cuda"))
    assert torch.equal(last, h0) and (dh == 1).all()
    y, last = M.gated_scan(torch.empty(2, 0, 5, device="cuda"), torch.empty(2, 0, 5, device="cuda"), [0, 4], h0=h0[:2])
    assert torch.equal(last, h0[:2])
    y, last = M.gated_scan(torch.empty(0, 4, 5, device="cuda"), torch.empty(0, 4, 5, device="cuda"))
    assert last.shape == (0, 5)
    st = torch.rand(2, 11, device="cuda")
    assert torch.equal(M.running_norm(torch.empty(0, 5, device="cuda"), [0, 0], state=st)[1], st)


def test_two_streams_and_a_waiting_one(M):
    """Calls on two streams at once keep out of each other's way; each uses its own temporaries."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    xs = [torch.randn(1, 30000, 39, generator=gen, device="cuda") for _ in range(2)]
    gs = [torch.randn(1, 30000, 39, generator=gen, device="cuda") for _ in range(2)]
    want = [(M.gated_scan(x, g, form="sigmoid"), M.running_norm(x)) for x, g in zip(xs, gs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append((M.gated_scan(xs[k], gs[k], form="sigmoid"), M.running_norm(xs[k])))
    torch.cuda.synchronize()
    for k in range(2):
        for a, b in got[k]:
            assert torch.equal(a[0], want[k][0][0]) and torch.equal(a[1], want[k][0][1])
            assert torch.equal(b[0], want[k][1][0]) and torch.equal(b[1], want[k][1][1])


@pytest.mark.parametrize("counts,d", [([300, 40, 0, 7], 39), ([12000], 64)])
def test_captured_training_step(M, counts, d):
    """The operators together, as a training step uses them -- normalised rows, dropout with a step counter on the
    device, the recurrence and its gradient -- captured once and replayed on new data, against eager calls."""
    lay = M.Layout.from_frame_counts("cuda", counts)
    n = sum(counts)
    gen = torch.Generator(device="cuda").manual_seed(5)
    feats = torch.randn(n, d, generator=gen, device="cuda") * 3 + 1
    gate = torch.randn(n, d, generator=gen, device="cuda").requires_grad_(True)
    h0 = torch.randn(len(counts), d, generator=gen, device="cuda").requires_grad_(True)
    gy = torch.randn(n, d, generator=gen, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def run():
        rows, state = M.running_norm(feats, lay, decay=0.99)
        x = M.feature_dropout(rows, 0.2, 77, step=step, per="sequence", frame_counts=lay).requires_grad_(True)
        y, last = M.gated_scan(x, gate, lay, h0=h0, form="sigmoid")
        return (y.detach(), last.detach(), state) + torch.autograd.grad(y, (x, gate, h0), gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = run()
        step += 1
    step.zero_()
    for k in range(3):
        with torch.no_grad():
            feats.copy_(torch.randn(n, d, generator=gen, device="cuda") * (k + 1) + k)
            gate.copy_(torch.randn(n, d, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert int(step) == k + 1
        step.fill_(k)
        for a, b in zip(static, run()):
            assert torch.equal(a, b)
        step.fill_(k + 1)
    with pytest.raises(ValueError):
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2):
            M.running_norm(feats, counts)


def test_ctc_batch_with_dropout(M):
    rng = np.random.default_rng(2)
    audios = [np.clip(rng.standard_normal(n) * 3000, -32768, 32767).astype(np.int16) for n in (16000, 4000, 23456)]
    plain, lens = M.ctc_feature_batch(audios)
    got, lens2 = M.ctc_feature_batch(audios, dropout=0.25, seed=9, step=4)
    assert np.array_equal(lens, lens2) and torch.equal(M.ctc_feature_batch(audios)[0], plain)
    at = 0
    keep = keep_mask((int(lens.sum()), 39), lens, "sequence", 0.25, 9, 4)
    for u, n in enumerate(lens):
        k = torch.from_numpy(keep[at:at + n]).cuda()
        at += n
        want = torch.where(k, plain[u, :n] * (1 / 0.75), 0.0)
        assert (got[u, :n] - want).abs().max() <= 3 * U * float(want.abs().max()) and not got[u, n:].any()
        assert torch.equal(got[u, :n] == 0, ~k | (plain[u, :n] == 0))
    # on to the padded recurrence, with the lengths as pad_sequences reports them
    y, last = M.gated_scan(got, torch.full_like(got, 2.0), lens, form="sigmoid")
    for u, n in enumerate(lens):
        assert torch.equal(y[u, n - 1], last[u])
    with pytest.raises(ValueError):
        M.ctc_feature_batch(audios, dropout=0.25)


def test_streaming_with_running_norm(M):
    """Rows of live streams normalised as they become final equal the normalised rows of the whole utterance."""
    rng = np.random.default_rng(3)
    audio = np.clip(rng.standard_normal((3, 16000)) * 3000, -32768, 32767).astype(np.int16)
    plain = M.StreamingMFCC("self5", n_streams=3, max_chunk=1600)
    s = M.StreamingMFCC("self5", n_streams=3, max_chunk=1600, running_norm=0.98)
    for utterance in range(2):      # the second one starts from the prior again
        rows, normed = [], []
        for a in range(0, 16000, 800):
            chunk = torch.from_numpy(audio[:, a:a + 800]).cuda()
            rows.append(plain.push(chunk).clone())
            normed.append(s.push(chunk).clone())
        rows.append(plain.flush().clone())
        normed.append(s.flush().clone())
        rows, normed = torch.cat(rows, 1), torch.cat(normed, 1)
        want, _ = M.running_norm(rows, decay=0.98)
        # both run the same sums in pieces: within 2 x 32 u X / sigma, X / sigma below 300 for these rows but the first
        assert normed.shape == want.shape and not normed[:, 0].any()
        assert (normed - want).abs().max() <= 64 * U * 300 * 4
    prior = M.running_norm_state(M.cmvn_accumulate(rows.reshape(-1, 39).contiguous()), 100.0)
    t = M.StreamingMFCC("self5", n_streams=3, max_chunk=16000, running_norm=0.98, norm_state=prior)
    parts = [t.push(torch.from_numpy(audio).cuda()).clone(), t.flush().clone()]
    want, _ = M.running_norm(rows, decay=0.98, state=prior.repeat(3, 1))
    assert (torch.cat(parts, 1) - want).abs().max() <= 64 * U * 300 * 4
    t.push(torch.from_numpy(audio[:, :4000]).cuda())
    t.reset()
    assert torch.equal(t.push(torch.from_numpy(audio).cuda()), parts[0])


# --------------------------------------------------------------------------
# the corners of the division over workgroups
# --------------------------------------------------------------------------
@pytest.mark.parametrize("counts,d", [([600, 13, 590] + [450] * 13, 512), ([700, 0, 3, 650], 257), ([30] * 40, 130), ([3, 20, 17, 1, 24] * 9, 5)])
def test_scan_divisions(M, counts, d):
    """Narrower column blocks for few sequences, several short sequences to a workgroup, several column blocks."""
    check_scan(M, counts, d, torch.float32, "sigmoid", seed=d)
    check_scan(M, counts, d, torch.bfloat16, "decay", reverse=True, seed=d, h0=False)


def test_norm_many_sequences(M):
    """So many sequences that workgroups take half the threads."""
    rng = np.random.default_rng(5)
    check_norm(M, [120] + rng.integers(0, 21, size=2100).tolist(), 39, 0.98, seed=2)


@pytest.mark.parametrize("n,k,d", [(64, 1, 39), (200, 3, 39), (40, 8, 13), (500, 5, 2)])
def test_short_sequences_in_place(M, n, k, d):
    """One slot of time to a sequence; threads without a slot of their own must not disturb the rows of others."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    x, g = torch.randn(n, k, d, generator=gen, device="cuda"), torch.rand(n, k, d, generator=gen, device="cuda")
    st = M.running_norm(torch.randn(n, 50, d, generator=gen, device="cuda"))[1]
    want_y, want_last = M.gated_scan(x, g, form="sigmoid")
    want_n, want_s = M.running_norm(x, state=st)
    for _ in range(20):
        a, b = x.clone(), x.clone()
        y, last = M.gated_scan(a, g, form="sigmoid", out=a)
        z, s = M.running_norm(b, state=st, out=b)
        assert torch.equal(a, want_y) and torch.equal(last, want_last) and torch.equal(b, want_n) and torch.equal(s, want_s)
    # y over the gates instead
    c = g.clone()
    M.gated_scan(x, c, form="sigmoid", out=c)
    assert torch.equal(c, want_y)


def test_rows_far_apart(M):
    """Row strides at which a tile spans more than 4 GiB."""
    n, d, ld = 220, 40, 10_500_000
    big = torch.empty(n * ld, device="cuda")
    far = big.as_strided((n, d), (ld, 1))
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, g, gy = (torch.randn(n, d, generator=gen, device="cuda") for _ in range(3))
    far.copy_(x)
    for reverse in (False, True):
        a, b = x.clone().requires_grad_(True), g.clone().requires_grad_(True)
        y, last = M.gated_scan(a, b, [200, 20], form="sigmoid", reverse=reverse)
        want = torch.autograd.grad((y, last), (a, b), (gy, torch.ones_like(last)))
        c, e = far.detach().requires_grad_(True), g.clone().requires_grad_(True)
        y2, last2 = M.gated_scan(c, e, [200, 20], form="sigmoid", reverse=reverse)
        got = torch.autograd.grad((y2, last2), (c, e), (gy, torch.ones_like(last)))
        assert torch.equal(y, y2) and torch.equal(last, last2) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    z, s = M.running_norm(x, [200, 20])
    z2, s2 = M.running_norm(far, [200, 20], out=far)
    assert z2 is far and torch.equal(z, far) and torch.equal(s, s2)
    far.copy_(x)
    for per in ("element", "frame", "sequence"):
        assert torch.equal(M.feature_dropout(far, 0.4, 5, per=per, frame_counts=[200, 20]), M.feature_dropout(x, 0.4, 5, per=per, frame_counts=[200, 20]))
    del big, far, z2, c, got


def test_more_than_2_31_values(M):
    n, d = 70000, 32768
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(n, d, generator=gen, device="cuda", dtype=torch.float16)
    g = torch.full((1, d), 3.0, device="cuda", dtype=torch.float16).expand(n, d)
    y, last = M.gated_scan(x, g, form="sigmoid")
    cols = [0, 1, 12345, d - 1]
    xs = host(x[:, cols])
    out, mag = sequence(xs, np.full_like(xs, 3.0), np.zeros(4), "sigmoid", False)
    close(y[:, cols], out[0], mag[0], torch.float16, memory(np.array([3.0]), "sigmoid", n), "y")
    close(last[0, cols], out[1], mag[1], torch.float32, memory(np.array([3.0]), "sigmoid", n), "last")
    M.feature_dropout(x, 0.3, 21, step=2, out=y)
    rows = [0, 1, 65535, n - 1]
    e = np.array(rows, dtype=np.uint64)[:, None] * np.uint64(d) + np.arange(d, dtype=np.uint64)
    keep = fields(e, 2, 21) >= int(round(0.3 * 65536))
    got, src = host(y[rows]), host(x[rows])
    assert np.array_equal(got == 0, ~keep | (src == 0))
    ref = src * keep * 65536 / (65536 - int(round(0.3 * 65536)))
    assert (np.abs(got - ref) <= (2 * U + HALF[torch.float16]) * np.abs(ref) + TINY[torch.float16]).all()
    del x, y


def test_not_rows(M):
    v = torch.zeros(8, device="cuda")
    for f in (lambda: M.gated_scan(v, v), lambda: M.gated_scan(v[0], v[0]), lambda: M.running_norm(v), lambda: M.feature_dropout(v, 0.5, 1),
              lambda: M.gated_scan_step(v, v, v), lambda: M.gated_scan(None, v), lambda: M.gated_scan(torch.zeros(3, 0, device="cuda"), torch.zeros(3, 0, device="cuda"))):
        with pytest.raises(ValueError):
            f()


def test_gradient_at_another_stream(M):
    """The backward pass runs on the stream of the forward pass, with the caller ordering the streams as usual."""
    x, g = torch.randn(5000, 64, device="cuda", requires_grad=True), torch.randn(5000, 64, device="cuda", requires_grad=True)
    y, last = M.gated_scan(x, g, form="sigmoid")
    want = torch.autograd.grad(y.sum() + last.sum(), (x, g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, last = M.gated_scan(x, g, form="sigmoid")
        loss = y.sum() + last.sum()
    torch.cuda.current_stream().wait_stream(side)
    got = torch.autograd.grad(loss, (x, g))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_padding_is_not_read_and_audio_layouts(M):
    gen = torch.Generator(device="cuda").manual_seed(7)
    lens = [40, 0, 300, 17, 299]
    for reverse in (False, True):
        x, g, gy = (torch.randn(5, 300, 39, generator=gen, device="cuda") for _ in range(3))
        runs = []
        for fill in (0.0, float("nan")):
            a, b, c = x.clone(), g.clone(), gy.clone()
            for u, n in enumerate(lens):
                for t in (a, b, c):
                    t[u, n:] = fill
            z, s = M.running_norm(a, lens)
            a.requires_grad_(True), b.requires_grad_(True)
            y, last = M.gated_scan(a, b, lens, form="sigmoid", reverse=reverse)
            runs.append((z, s, y.detach(), last.detach()) + torch.autograd.grad(y, (a, b), c))
        for p, q in zip(*runs):
            assert torch.equal(p, q) and torch.isfinite(p).all()
    # the layout that cut the audio also tells the sequences of its rows
    fe = M.MFCC("self5")
    rng = np.random.default_rng(1)
    lengths = [16000, 4000, 23456]
    audio = torch.from_numpy(np.clip(rng.standard_normal(sum(lengths)) * 3000, -32768, 32767).astype(np.int16)).cuda()
    lay = fe.layout(lengths)
    feats = fe.forward(audio, lay)
    counts = np.diff(lay.frame_offsets)
    assert torch.equal(M.running_norm(feats, lay)[0], M.running_norm(feats, counts)[0])
    assert torch.equal(M.gated_scan(feats, torch.sigmoid(feats), lay)[0], M.gated_scan(feats, torch.sigmoid(feats), torch.from_numpy(counts))[0])
    assert torch.equal(M.feature_dropout(feats, 0.5, 1, per="sequence", frame_counts=lay), M.feature_dropout(feats, 0.5, 1, per="sequence", frame_counts=counts))


@pytest.mark.parametrize("what", ["scan", "step", "step state", "norm", "norm state", "dropout"])
def test_written_tensors_count_as_changed(M, what):
    """A tensor that a product saved for its backward pass, then written as out= / state_out=: an error, no wrong gradient."""
    d = 6
    x, g, h = (torch.rand(5, d, device="cuda") for _ in range(3))
    w = torch.ones((1, 1 + 2 * d) if what == "norm state" else (5, d), device="cuda", requires_grad=True)
    t = torch.rand(w.shape, device="cuda")
    loss = (w * t).sum()
    calls = {"scan": lambda t: M.gated_scan(x, g, out=t), "step": lambda t: M.gated_scan_step(x, g, h, out=t),
             "step state": lambda t: M.gated_scan_step(x, g, h, state_out=t), "norm": lambda t: M.running_norm(x, out=t),
             "norm state": lambda t: M.running_norm(x, state_out=t), "dropout": lambda t: M.feature_dropout(x, 0.5, 1, out=t)}
    calls[what](t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.no_grad(), pytest.raises(ValueError, match="requires a gradient"):
        calls[what](w)
    with torch.inference_mode():
        calls[what](torch.rand(w.shape, device="cuda"))
