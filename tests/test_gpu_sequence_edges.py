"""Corners of the operators along time on the device: last column blocks of few groups, tensors that overlap, values and gates at
the ends of their range.  Definitions and tolerances are those of test_gpu_sequence_ops.py."""
import numpy as np
import pytest
import torch

from test_gpu_sequence_ops import HALF, TINY, M, U, check_norm, check_scan, host, make_gate, memory, norm_sequence, sequence  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,d", [([300, 40], 807), ([100, 7], 869), ([300] * 3, 993), ([100, 0, 250], 1025), ([300] * 15, 1025), ([90, 120], 1285),
                                      ([60, 9], 1799), ([300, 5], 2050), ([8] * 64, 3655), ([900], 4097)])
def test_norm_last_column_block(M, counts, d):
    """Widths whose last block of columns has fewer groups than a slot has rows; every sequence has a weight of its own."""
    check_norm(M, counts, d, 0.97, seed=d)
    x, y, end = check_norm(M, counts, d, 1.0, dtype=torch.bfloat16, state=False, seed=d)
    z = x.clone()
    y, end = M.running_norm(x, counts, decay=0.97)
    assert torch.equal(M.running_norm(z, counts, decay=0.97, out=z)[1], end) and torch.equal(z, y)


@pytest.mark.parametrize("counts,d", [([70, 9], 1025), ([200], 807), ([70, 30], 2050)])
def test_scan_last_column_block(M, counts, d):
    check_scan(M, counts, d, torch.float32, "sigmoid", seed=d)
    check_scan(M, counts, d, torch.bfloat16, "decay", reverse=True, seed=d)


def test_forward_mode_is_refused(M):
    """Dual tensors do not require a gradient; every call refuses them instead of returning a value without its tangent."""
    x, g, h = (torch.rand(5, 6, device="cuda") for _ in range(3))
    st = torch.rand(1, 13, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: M.gated_scan(dual(x), g), lambda: M.gated_scan(x, dual(g)), lambda: M.gated_scan(x, g, h0=dual(h[:1])),
                 lambda: M.gated_scan(x.clone().requires_grad_(True), dual(g)), lambda: M.gated_scan(x, g, out=dual(h.clone())),
                 lambda: M.gated_scan_step(x, g, dual(h)), lambda: M.gated_scan_step(dual(x), g, h), lambda: M.gated_scan_step(x, g, h, state_out=dual(h)),
                 lambda: M.running_norm(dual(x)), lambda: M.running_norm(x, state=dual(st)), lambda: M.running_norm(x, out=dual(h.clone())),
                 lambda: M.feature_dropout(dual(x), 0.5, 1), lambda: M.feature_dropout(x, 0.5, 1, out=dual(h.clone()))]
        for call in calls:
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(ValueError, match="tangent"):
                    call()
        assert torch.equal(M.gated_scan(x, g)[0], M.gated_scan(x, g)[0])    # tensors without one go on as ever


def test_overlap_is_refused(M):
    from mfcc_amd import _capi as capi
    buf = torch.rand(2, 21, 8, device="cuda")
    x, g = buf[:, :20], torch.rand(2, 20, 8, device="cuda")
    st = torch.zeros(3, 17, device="cuda")
    h = torch.zeros(3, 8, device="cuda")
    for f in (lambda: M.gated_scan(x, g, out=buf[:, 1:]), lambda: M.gated_scan(g, x, out=buf[:, 1:]), lambda: M.running_norm(x, out=buf[:, 1:]),
              lambda: M.running_norm(x, state=st[:2], state_out=st[1:]), lambda: M.running_norm(x, state=st[1:], state_out=st[:2]),
              lambda: M.feature_dropout(x, 0.5, 1, out=buf[:, 1:]), lambda: M.gated_scan_step(g[0, :2], g[1, :2], h[:2], state_out=h[1:]),
              lambda: M.gated_scan_step(buf[0, :2], g[1, :2], h[:2], out=buf[0, 1:3])):
        with pytest.raises(capi.MfccError, match="overlaps"):
            f()
    wide = torch.rand(2, 20, 24, device="cuda")       # parts of the same rows do not
    a, b, c = wide[..., :8], wide[..., 8:16], wide[..., 16:]
    want = M.gated_scan(a, b)[0]
    assert torch.equal(M.gated_scan(a, b, out=c)[0], want) and torch.equal(M.gated_scan(a, b, out=b)[0], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", ["decay", "sigmoid"])
@pytest.mark.parametrize("reverse", [False, True])
def test_infinities_over_pieces(M, dtype, form, reverse):
    """Long sequences: an infinity stays one over pieces whose products of gates vanish in 32 bits, forwards and backwards."""
    n, d = 9000, 64
    gen = torch.Generator(device="cuda").manual_seed(11)
    x, gy = (torch.randn(n, d, generator=gen, device="cuda").to(dtype) for _ in range(2))
    g = make_gate(gen, (n, d), form, dtype)
    g[g == 0] = 0.5
    x[4000, 1], x[100, 2], x[8900, 3] = float("inf"), -float("inf"), float("inf")
    gy[5000, 4], gy[8990, 5] = float("inf"), -float("inf")
    h0, gl = (torch.randn(1, d, generator=gen, device="cuda") for _ in range(2))
    h0[0, 6] = float("inf")
    leaves = [t.requires_grad_(True) for t in (x, g, h0)]
    y, last = M.gated_scan(x, g, [n], h0=h0, form=form, reverse=reverse)
    dx, _, dh = torch.autograd.grad((y, last), leaves, (gy, gl))
    with np.errstate(invalid="ignore"):
        out, mag = sequence(host(x), host(g), host(h0)[0], form, reverse, host(gy), host(gl)[0])
    mem = memory(host(g), form, n)
    for got, ref, m, dt, what in ((y, out[0], mag[0], dtype, "y"), (last[0], out[1], mag[1], torch.float32, "last"), (dx, out[2], mag[2], dtype, "dx"),
                                  (dh[0], out[4], mag[4], torch.float32, "dh0")):
        got, fin = host(got), np.isfinite(ref)
        assert (~fin).any() or reverse, what
        assert np.array_equal(got[~fin], ref[~fin]), what
        tol = 16 * U * (1 + mem) * m[fin] + HALF[dt] * np.abs(ref[fin]) + TINY[dt]
        assert (np.abs(got[fin] - ref[fin]) <= tol).all(), what


def test_products_of_gates_past_32_bits(M):
    n, d = 9000, 64
    x = torch.randn(n, d, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    g = torch.full((n, d), 0.9, device="cuda")
    g[:6000, :4] = 1.1
    x[:5900, 0] = 0              # nothing there to grow until shortly before the gates fall
    x[:6000, 1], g[6000, 1] = 0, 0
    g[:6001:500, 2] = 0          # 1.1 ** 500 = 5e20 in between
    g[:6000, 3], x[:6000, 3] = -1.1, 0
    y, last = M.gated_scan(x, g, [n])
    out, mag = sequence(host(x), host(g), np.zeros(d), "decay", False)
    assert np.isfinite(out[0]).all()
    for got, ref, m in ((y, out[0], mag[0]), (last[0], out[1], mag[1])):
        assert (np.abs(host(got) - ref) <= 16 * U * (1 + n) * m).all()


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -149, 2.0 ** -127])
def test_norm_of_subnormal_variances(M, eps):
    """Variances around the smallest normal number without an eps that covers them."""
    from test_sequence_kernels_cpu import norm_definition, small_variance_tolerance, small_variances
    rng, n, d, decay = np.random.default_rng(5), 300, 24, 0.9
    x = small_variances(rng, n, d)
    y = M.running_norm(torch.from_numpy(x).cuda(), decay=decay, eps=eps)[0]
    with np.errstate(invalid="ignore"):
        ref, fin, _ = norm_definition(x.astype(np.float64), decay, np.zeros(1 + 2 * d), eps)
    tol, known = small_variance_tolerance(x.astype(np.float64), ref, decay, fin)
    known[0] = False
    assert known.mean() > 0.5 and (np.abs(host(y) - ref)[known] <= tol[known] + 32 * U * 8).all()   # means of values below 8 sigma


def test_norm_from_a_state_without_weight(M):
    """A prior of weight 0 is no prior, wherever its means are: as a state, over pieces, and in live streams."""
    rng = np.random.default_rng(7)
    for n in (1, 5, 40, 9000):
        x = torch.from_numpy((rng.standard_normal((n, 39)) * 3 + 7).astype(np.float32)).cuda()
        st = torch.zeros(1, 79, device="cuda")
        st[:, 1:40] = torch.from_numpy(rng.standard_normal(39) * 1000)
        y, end = M.running_norm(x, state=st)
        want, fin = M.running_norm(x)
        assert torch.equal(y, want) and torch.equal(end, fin)
    sums = torch.cat([torch.tensor([50.0]), torch.full((39,), 5e4), torch.full((39,), 6e7)]).double().cuda()     # means of 1000
    audio = torch.from_numpy((rng.standard_normal((2, 8000)) * 3000).astype(np.int16)).cuda()
    a = M.StreamingMFCC("self5", n_streams=2, max_chunk=8000, running_norm=0.98)
    b = M.StreamingMFCC("self5", n_streams=2, max_chunk=8000, running_norm=0.98, norm_state=M.running_norm_state(sums, 0.0))
    assert torch.equal(a.push(audio), b.push(audio)) and torch.equal(a.flush(), b.flush())


def time_major(*shape, dtype=torch.float32):
    """[B, T, D] whose memory runs over the sequences first"""
    b, t, d = shape
    return torch.empty(t, b, d, dtype=dtype, device="cuda").transpose(0, 1)


@pytest.mark.parametrize("d", [39, 40, 257])
@pytest.mark.parametrize("counts", [None, [30, 0, 17, 90, 5]])
def test_orders_of_rows(M, d, counts):
    """Inputs and outputs in time-major memory and between other columns give the bits of rows one after the other."""
    gen = torch.Generator(device="cuda").manual_seed(d)
    x, g, gy = (torch.randn(5, 70, d, generator=gen, device="cuda") for _ in range(3))
    xt, gt, gyt = (time_major(5, 70, d).copy_(t) for t in (x, g, gy))
    wide = torch.full((5, 70, d + 9), 7.0, device="cuda")

    def places(dtype):
        yield time_major(5, 70, d, dtype=dtype)
        w = wide.to(dtype)
        yield w[..., 3:3 + d]
        assert (w[..., :3] == 7).all() and (w[..., 3 + d:] == 7).all()

    for dtype in (torch.float32, torch.bfloat16):
        z, s = M.running_norm(x, counts, dtype=dtype)
        for out in places(dtype):
            z2, s2 = M.running_norm(xt, counts, out=out)
            assert z2 is out and torch.equal(z2, z) and torch.equal(s2, s)
        xd = x.to(dtype)
        for per in ("element", "frame", "sequence"):
            want = M.feature_dropout(xd, 0.4, 5, per=per, frame_counts=counts)
            for out in places(dtype):
                assert torch.equal(M.feature_dropout(xt.to(dtype), 0.4, 5, per=per, frame_counts=counts, out=out), want)
                assert torch.equal(M.feature_dropout(out.copy_(xd), 0.4, 5, per=per, frame_counts=counts, out=out), want)
        gd = g.to(dtype)
        want, last = M.gated_scan(xd, gd, counts, form="sigmoid", reverse=True)
        for out in places(dtype):
            assert torch.equal(M.gated_scan(xt.to(dtype), gt.to(dtype), counts, form="sigmoid", reverse=True, out=out)[0], want)
    grads = []
    for a, b, c in ((x, g, gy), (xt, gt, gyt)):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y, last = M.gated_scan(a, b, counts, form="sigmoid")
        grads.append((y.detach(), last.detach()) + torch.autograd.grad(y, (a, b), c))
    assert all(torch.equal(p, q) for p, q in zip(*grads))
    xr = xt.detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(M.feature_dropout(xr, 0.4, 5, per="sequence"), xr, gyt)
    assert torch.equal(dx, M.feature_dropout(gy, 0.4, 5, per="sequence"))
