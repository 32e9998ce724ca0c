"""Calls that the sequence operators refuse before they look for a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fw


def calls(x, w):
    """Each operator on x (2, 3, 4) and w (5, 4)."""
    import videometamaterials_amd as vm
    return (lambda: vm.gated_linear_scan(x, x), lambda: vm.gated_linear_scan(x.detach(), x.detach(), x[:, 0]), lambda: vm.gated_feed_forward(x, w, w),
            lambda: vm.gated_feed_forward(x, w, w, w[:, 0].contiguous(), w[:, 0].contiguous()), lambda: vm.grad_norm([w]), lambda: vm.clip_grad_norm_([x, w], 1.0))


def test_forward_mode_derivatives():
    """The output would come back without a tangent, that is with a derivative of zero."""
    x, w = torch.zeros(2, 3, 4), torch.zeros(5, 4)
    with fw.dual_level():
        for a, b in ((fw.make_dual(x, x), w), (x, fw.make_dual(w, w)), (fw.make_dual(x, x), fw.make_dual(w, w))):
            duals = [a is not x, a is not x, True, True, b is not w, True]
            for call, refused in zip(calls(a, b), duals):
                if refused:
                    with pytest.raises(NotImplementedError, match="forward"):
                        call()
