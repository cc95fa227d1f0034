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
