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


def test_tracing():
    """A trace would hold the empty output alone, and its replay return memory that nobody wrote."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = torch.zeros(2, 3, 4), torch.zeros(5, 4)
    for k in range(6):
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(lambda x, w: calls(x, w)[k](), (x, w))
        for pre in (False, True):
            with pytest.raises(NotImplementedError, match="traced"):
                make_fx(lambda x, w: calls(x, w)[k](), pre_dispatch=pre)(x, w)
        with FakeTensorMode(), pytest.raises(NotImplementedError, match="traced"):
            calls(torch.zeros(2, 3, 4), torch.zeros(5, 4))[k]()


def test_tensors_that_stand_in_for_others():
    class Wrapped(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError("reached")
    x, w = torch.zeros(2, 3, 4), torch.zeros(5, 4)
    negative = torch.zeros(2, 3, 4, dtype=torch.complex64).conj().imag
    assert negative.is_neg()
    from videometamaterials_amd import gated_feed_forward, gated_linear_scan, grad_norm
    for a in (Wrapped(x), negative):
        for call in (lambda: gated_linear_scan(a, x), lambda: gated_linear_scan(x, a), lambda: gated_feed_forward(a, w, w), lambda: grad_norm([a])):
            with pytest.raises(NotImplementedError, match="plain"):
                call()
    for k in range(6):
        with pytest.raises(NotImplementedError, match="plain"):
            torch.func.vmap(lambda x, w: calls(x, w)[k]())(x[None], w[None])
        with pytest.raises(NotImplementedError, match="plain"):
            torch.func.grad(lambda x: calls(x, x[0, :, :])[k]().sum())(x)
    assert isinstance(torch.nn.Parameter(x), torch.Tensor)
    with pytest.raises(Exception, match="GPU"):  # a parameter is a plain tensor
        gated_feed_forward(x, torch.nn.Parameter(w), w)
