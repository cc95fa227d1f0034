"""What the Python side of the operators along time decides on the host, without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

recurrent = pytest.importorskip("mfcc_amd.recurrent")


def test_tangents_are_seen():
    x, t = torch.randn(3, 4), torch.ones(3, 4)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        recurrent._no_tangent(x, None, 3)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(ValueError, match="tangent"):
                recurrent._no_tangent(x, None, dual)
        recurrent._no_tangent(forward_ad.unpack_dual(dual).primal)
        with torch.inference_mode():     # nothing is differentiated there, in any mode
            recurrent._no_tangent(dual)
    recurrent._no_tangent(x)


def test_state_from_sums_of_no_rows():
    """An accumulator that has seen nothing is no prior, whatever weight it is given."""
    for weight in (0.0, 50.0):
        assert recurrent.running_norm_state(torch.zeros(7, dtype=torch.float64), weight, 2).tolist() == [[0.0] * 7] * 2
    sums = torch.tensor([4.0, 8.0, -4.0, 20.0, 4.0], dtype=torch.float64)
    assert recurrent.running_norm_state(sums, 10.0).tolist() == [[10.0, 2.0, -1.0, 10.0, 0.0]]
    assert recurrent.running_norm_state(sums, 0.0).tolist() == [[0.0, 2.0, -1.0, 0.0, 0.0]]
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            recurrent.running_norm_state(sums, bad)
