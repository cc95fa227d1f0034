"""Corners of the operators along time on the device: last column blocks of few groups, tensors that overlap, values and gates at
the ends of their range.  Definitions and tolerances are those of test_gpu_sequence_ops.py."""
import numpy as np
import pytest
import torch

from test_gpu_sequence_ops import M, U, check_norm, check_scan, host, norm_sequence  # noqa: F401

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
