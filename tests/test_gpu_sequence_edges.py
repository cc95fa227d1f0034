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
