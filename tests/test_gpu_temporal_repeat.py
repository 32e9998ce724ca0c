"""The fused temporal block gives the same bits at every launch, with and without tokens, in each of its modes."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


def packed(N, lib, w, fmt):
    """(out, in) weight as fragments for vmm_temporal_block_*."""
    co, ci = w.shape
    out = torch.zeros((co + 31) // 32 * 32 * ((ci + 31) // 32 * 32), device=w.device)
    job = (N.PackJob * 1)()
    j = job[0]
    j.torch_w, j.packed = w.data_ptr(), out.data_ptr()
    j.TH, j.TW, j.C, j.Cp, j.N = 1, 1, ci, ci, co
    j.sn, j.sc, j.fmt = ci, 1, fmt
    table = torch.frombuffer(bytearray(bytes(job)), dtype=torch.uint8).to(w.device)
    N.check(lib.vmm_pack_weights(table.data_ptr(), 1, out.numel(), 0, torch.cuda.current_stream().cuda_stream), "pack")
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("channels,T,HW", [(64, 5, 256), (64, 11, 144), (64, 22, 49), (128, 5, 256), (128, 11, 64)])
@pytest.mark.parametrize("ntok", [0, 5])
def test_same_bits_at_every_launch(gpu, channels, T, HW, ntok):
    from videometamaterials_amd import _native as N, hostmath
    lib = N.lib()
    B, heads, hid = 3, 8, 256
    g = torch.Generator(device=gpu).manual_seed(T)
    n = lambda *s, k=1.0: torch.randn(*s, generator=g, device=gpu) * k  # noqa: E731
    x, gamma, bias = n(B * T * HW, channels), 1 + n(channels, k=0.2), n(heads, T, T)
    wqkv, wout = n(3 * hid, channels, k=0.125), n(channels, hid, k=0.0625)
    ek, ev = (n(B, ntok, hid), n(B, ntok, hid)) if ntok else (None, None)
    rot = hostmath.rotary_table(T, 32).to(gpu)
    first = {}
    for name, fmt in (("bf16x3", 0), ("bf16", 0), ("fp16", 16)):
        wq, wo = packed(N, lib, wqkv, 2 | fmt), packed(N, lib, wout, 3 | fmt)
        out = torch.empty_like(x)
        for launch in range(6):
            out.fill_(7.0)
            N.check(getattr(lib, "vmm_temporal_block_" + name)(
                x.data_ptr(), channels, gamma.data_ptr(), wq.data_ptr(), wo.data_ptr(), ek.data_ptr() if ntok else None, ev.data_ptr() if ntok else None, ntok,
                bias.data_ptr(), 0, rot.data_ptr(), out.data_ptr(), channels, B, T, HW, channels, heads, C.c_float(32 ** -0.5), C.c_float(1e-5),
                torch.cuda.current_stream().cuda_stream), name)
            assert torch.equal(first.setdefault(name, out.clone()), out), (name, launch)
    # the modes are the same block; of eight operands (rows, weights, q, k, v, softmax, its product, weights) each is off by half a step of its type at most
    branch = first["bf16x3"] - x
    for name, bits in (("bf16", 8), ("fp16", 11)):
        assert float((first[name] - x - branch).norm() / branch.norm()) < 8 * 2.0 ** -bits, name
