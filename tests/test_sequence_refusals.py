"""Calls that the sequence operators refuse before they look for a GPU."""
import ctypes as C

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


def test_a_workspace_that_is_too_small_is_refused():
    """Sizes depend on more than sizes: alignment, strides, which buffers are there.  A query without them gives less than the call needs; the call says so."""
    from videometamaterials_amd import _native as N
    lib = N.lib()
    a = [(k + 1) << 24 for k in range(12)]

    def refused(call, query, desc, backward, less):
        need = query(C.byref(desc), backward)
        assert need > less >= 0
        desc.workspace = 1 << 30
        for size in {0, less, need - 1}:
            desc.workspace_bytes = size
            assert call(C.byref(desc), None) == -1
    scan = dict(x=a[0], x_row=8, gate=a[1], gate_row=8, y=a[2], y_row=8, B=2, D=8, type=1)
    kept = N.GatedScanDesc(**scan, L=1000, states=a[3])
    refused(lib.vmm_gated_scan, lib.vmm_gated_scan_workspace, N.GatedScanDesc(**scan, L=1000), 0, lib.vmm_gated_scan_workspace(C.byref(kept), 0))
    refused(lib.vmm_gated_scan_bwd, lib.vmm_gated_scan_workspace, N.GatedScanDesc(**scan, L=1000, states=a[3]), 1, lib.vmm_gated_scan_workspace(C.byref(kept), 0))
    ff = dict(x=a[0], ldx=40, w_gate=a[1], w_up=a[2], h=a[3], ldh=64, M=64, K=40, F=64, type=1)
    bare = lib.vmm_gated_ff_workspace(C.byref(N.GatedFFDesc(M=64, K=40, F=64, type=1, ldx=40)), 0)  # nothing but sizes
    for odd in (dict(x=a[0] + 2), dict(w_gate=a[1] + 2), dict(w_up=a[2] + 8), dict(ldx=41)):
        refused(lib.vmm_gated_ff, lib.vmm_gated_ff_workspace, N.GatedFFDesc(**dict(ff, **odd)), 0, bare)
    back = dict(ff, M=600, F=1024, g_pre=a[4], u_pre=a[5], dh=a[6], lddh=1024)
    for wanted in (dict(dx=a[7], lddx=40), dict(dw_gate=a[8], dw_up=a[9])):
        refused(lib.vmm_gated_ff_bwd, lib.vmm_gated_ff_workspace, N.GatedFFDesc(**back, **wanted), 1, lib.vmm_gated_ff_workspace(C.byref(N.GatedFFDesc(**back)), 1))


@pytest.mark.parametrize("name", ["ldx", "ldh", "lddh", "lddx"])
@pytest.mark.parametrize("value", [-1, -8, 1 << 22])
def test_leading_dimensions_of_the_feed_forward_product(name, value):
    """A negative one would be read in front of its buffer."""
    from videometamaterials_amd import _native as N
    lib = N.lib()
    a = [(k + 1) << 24 for k in range(12)]
    d = N.GatedFFDesc(**dict(x=a[0], ldx=8, w_gate=a[1], w_up=a[2], h=a[3], ldh=8, g_pre=a[4], u_pre=a[5], dh=a[6], lddh=8, dx=a[7], lddx=8, M=4, K=8, F=8, type=1,
                             workspace=1 << 30, workspace_bytes=1 << 30) | {name: value})
    assert lib.vmm_gated_ff_workspace(C.byref(d), 0) == -1 and lib.vmm_gated_ff_workspace(C.byref(d), 1) == -1
    assert lib.vmm_gated_ff(C.byref(d), None) == -1 and lib.vmm_gated_ff_bwd(C.byref(d), None) == -1


@pytest.mark.parametrize("bound", [0.0, -1.0, float("nan"), 1e-46, 2.0 ** -151])
def test_bounds_that_are_no_positive_float32(bound):
    """2^-151 becomes zero in float32, and zero means that nothing is clipped."""
    import videometamaterials_amd as vm
    from videometamaterials_amd.dp import DataParallelTrainer
    for call in (lambda: vm.clip_grad_norm_([], bound), lambda: vm.ClippedAdam([torch.zeros(3)], max_norm=bound), lambda: DataParallelTrainer(None, max_grad_norm=bound)):
        with pytest.raises(ValueError, match="positive"):
            call()
    assert float(vm.clip_grad_norm_([], 2.0 ** -149)) == 0.0
