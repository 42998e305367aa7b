"""Forward-mode tangents: operators without a derivative refuse inputs that carry one, as they refuse
inputs that ask for a gradient (CPU only: the check is made before any GPU work)."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from musc_hip import _runtime as rt


def test_dual_tensors_are_refused():
    x = torch.ones(3)
    rt.require_no_gradient(x, None)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones(3))
        rt.require_no_gradient(x, None)
        with pytest.raises(ValueError, match='derivative|backward'):
            rt.require_no_gradient(None, x, dual)
        with torch.no_grad():                       # which leaves forward mode on
            with pytest.raises(ValueError, match='derivative|backward'):
                rt.require_no_gradient(dual)
        with torch.inference_mode():                # which does not
            rt.require_no_gradient(x)
        rt.require_no_gradient(fw.unpack_dual(dual).primal)
    rt.require_no_gradient(x)


def test_gradients_are_refused_as_before():
    leaf = torch.ones(3, requires_grad=True)
    with pytest.raises(ValueError, match='backward'):
        rt.require_no_gradient(torch.ones(3), leaf)
    with torch.no_grad():
        rt.require_no_gradient(leaf)
    rt.require_no_gradient(leaf.detach())
