"""Host side of the sequence operators: struct layouts, refusals that need no GPU, size queries."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_structs_match_the_header(tmp_path):
    from videometamaterials_amd import _native as N
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    pairs = {"vmm_gated_scan_desc": N.GatedScanDesc, "vmm_gated_ff_desc": N.GatedFFDesc, "vmm_grad_job": N.GradJob, "vmm_clip_adam_job": N.ClipAdamJob}
    hdr = open(os.path.join(ROOT, "include", "vmm_sequence.h")).read()
    assert set(re.findall(r"typedef struct (\w+)", hdr)) == set(pairs)
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "vmm_sequence.h"', "int main(void) {"]
    for name, cls in pairs.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, cls in pairs.items():
        assert int(got[name]) == C.sizeof(cls)
        assert all(int(got[f"{name}.{f}"]) == getattr(cls, f).offset for f, _ in cls._fields_)
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), hdr, flags=re.S).group(1), flags=re.S)
        assert len([m for decl in body.split(";") for m in decl.split(",") if m.strip()]) == len(cls._fields_)


def test_bad_descriptors_are_refused_before_any_launch():
    from videometamaterials_amd import _native as N
    lib = N.lib()
    ok = dict(x=1 << 20, x_row=4, gate=1 << 21, gate_row=4, y=1 << 22, y_row=4, L=200, B=1, D=4, type=0)
    assert lib.vmm_gated_scan(None, None) == -1 and lib.vmm_gated_scan_bwd(None, None) == -1
    for bad in (dict(type=3), dict(type=-1), dict(L=-1), dict(L=1 << 31), dict(B=-1), dict(D=-1), dict(B=1 << 16, D=1 << 16), dict(x_row=-1), dict(x_row=1 << 23),
                dict(dgate_row=-4), dict(B=1 << 22, L=256), dict(B=1 << 23, L=129), dict(B=1 << 24, L=1), dict(x=None), dict(gate=None), dict(y=None)):
        d = N.GatedScanDesc(**dict(ok, **bad))
        assert lib.vmm_gated_scan(C.byref(d), None) == -1, bad
        if not set(bad) & {"x", "gate", "y"}:
            assert lib.vmm_gated_scan_workspace(C.byref(d), 0) == -1 and lib.vmm_gated_scan_states(C.byref(d)) == -1
    d = N.GatedScanDesc(**ok)
    assert lib.vmm_gated_scan_workspace(C.byref(d), 0) > 0 and lib.vmm_gated_scan_states(C.byref(d)) == 4 * 4
    assert lib.vmm_gated_scan(C.byref(d), None) == -1  # more than one unit and no workspace
    d.workspace = 8
    assert lib.vmm_gated_scan(C.byref(d), None) == -1  # and one that is not aligned
    assert lib.vmm_gated_scan_bwd(C.byref(d), None) == -1  # no states
    d = N.GatedScanDesc(**dict(ok, L=64))
    assert lib.vmm_gated_scan_workspace(C.byref(d), 0) == 0 and lib.vmm_gated_scan_workspace(C.byref(d), 1) == 0
    for empty in (dict(B=0), dict(D=0)):
        assert lib.vmm_gated_scan(C.byref(N.GatedScanDesc(**dict(ok, **empty))), None) == 0

    ok = dict(x=1 << 20, ldx=8, w_gate=1 << 21, w_up=1 << 22, h=1 << 23, ldh=8, M=4, K=8, F=8, type=1)
    assert lib.vmm_gated_ff(None, None) == -1 and lib.vmm_gated_ff_bwd(None, None) == -1
    for bad in (dict(type=3), dict(act=2), dict(act=-1), dict(M=-1), dict(M=1 << 31), dict(K=0), dict(F=0), dict(K=1 << 22), dict(ldx=-1), dict(ldh=1 << 22), dict(M=(1 << 31) - 1, F=256)):
        d = N.GatedFFDesc(**dict(ok, **bad))
        assert lib.vmm_gated_ff(C.byref(d), None) == -1 and lib.vmm_gated_ff_workspace(C.byref(d), 0) == -1, bad
    for bad in (dict(x=None), dict(w_up=None), dict(h=None), dict(g_pre=1 << 24)):  # (one of the two kept tensors alone)
        assert lib.vmm_gated_ff(C.byref(N.GatedFFDesc(**dict(ok, **bad))), None) == -1, bad
    assert lib.vmm_gated_ff(C.byref(N.GatedFFDesc(**dict(ok, M=0))), None) == 0
    for t in range(3):  # no rows: sizes are still to be had
        assert lib.vmm_gated_ff_workspace(C.byref(N.GatedFFDesc(**dict(ok, M=0, type=t))), 0) >= 0 and lib.vmm_gated_ff_workspace(C.byref(N.GatedFFDesc(**dict(ok, M=0, type=t))), 1) >= 0
    d = N.GatedFFDesc(**dict(ok, type=0))
    assert lib.vmm_gated_ff_workspace(C.byref(d), 0) > 0 and lib.vmm_gated_ff(C.byref(d), None) == -1  # no workspace
    d = N.GatedFFDesc(**dict(ok, dh=1 << 24, lddh=8, g_pre=1 << 25, u_pre=1 << 26, dw_gate=1 << 27))
    assert lib.vmm_gated_ff_bwd(C.byref(d), None) == -1  # one weight gradient alone

    jobs = (N.GradJob * 2)(N.GradJob(1 << 20, 4, 0, 0), N.GradJob((1 << 20) + 8, 4, 0, 0))
    assert lib.vmm_grad_norm_workspace(jobs, 2) == 16 and lib.vmm_grad_norm_workspace(jobs, 0) == 8
    assert lib.vmm_grad_clip(jobs, 2, 1 << 21, None) == -2  # overlapping
    for bad in (N.GradJob(1 << 20, -1, 0, 0), N.GradJob(None, 4, 0, 0), N.GradJob((1 << 20) + 2, 4, 0, 0), N.GradJob(1 << 20, 4, 3, 0)):
        one = (N.GradJob * 1)(bad)
        assert lib.vmm_grad_norm_workspace(one, 1) == -1 and lib.vmm_grad_clip(one, 1, 1 << 21, None) == -1
        assert lib.vmm_grad_norm(one, 1, 1.0, 1.0, None, 1 << 21, 1 << 22, None) == -1
    a = 1 << 20
    for jobs_, want in (([(a, a + 64, a + 128, a + 64)], -2), ([(a, a + 64, a + 128, a + 192), (a + 8, a + 256, a + 320, a + 384)], -2), ([(a, a + 64, None, a + 128)], -1)):
        arr = (N.ClipAdamJob * len(jobs_))(*[N.ClipAdamJob(p, g, m, v, 4, 0, 0) for p, g, m, v in jobs_])
        assert lib.vmm_adam_step_clipped(arr, len(jobs_), 1e-3, 0.9, 0.999, 1e-8, 1, 1.0, 1 << 22, None, None) == want
    good = (N.ClipAdamJob * 1)(N.ClipAdamJob(a, a + 64, a + 128, a + 192, 4, 0, 0))
    assert lib.vmm_adam_step_clipped(good, 1, 1e-3, 0.9, 0.999, 1e-8, 0, 1.0, 1 << 22, None, None) == -1  # steps count from one


def test_host_tensors_and_unfit_arguments_are_refused():
    import videometamaterials_amd as vm
    from videometamaterials_amd._native import NativeError
    x = torch.zeros(2, 3, 4)
    with pytest.raises(NativeError):
        vm.gated_linear_scan(x, x)
    with pytest.raises(ValueError):
        vm.gated_linear_scan(x, x[:, :2])
    with pytest.raises(ValueError):
        vm.gated_linear_scan(x[0], x[0])
    for a, b in ((x, x.half()), (x.double(), x.double()), (x.int(), x.int())):
        with pytest.raises(TypeError):
            vm.gated_linear_scan(a, b)
    w, b = torch.zeros(5, 4), torch.zeros(5)
    with pytest.raises(NativeError):
        vm.gated_feed_forward(x, w, w)
    for args, kw in (((x, w[:, :3], w[:, :3]), {}), ((x, w, w[:4]), {}), ((x, w, w, b), {}), ((x, w, w, b, b[:4]), {}), ((x, w, w), dict(activation="relu")),
                     ((x, torch.zeros(0, 4), torch.zeros(0, 4)), {})):
        with pytest.raises(ValueError):
            vm.gated_feed_forward(*args, **kw)
    with pytest.raises(TypeError):
        vm.gated_feed_forward(x, w.half(), w)
    with pytest.raises(NativeError):
        vm.grad_norm([b])
    with pytest.raises(TypeError):
        vm.grad_norm([b.double()])
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            vm.clip_grad_norm_([b], bad)
    assert float(vm.grad_norm([])) == 0.0 and float(vm.clip_grad_norm_([], 1.0)) == 0.0
    with pytest.raises(NativeError):
        vm.ClippedAdam([b])
    for kw in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(max_norm=0.0), dict(step=-1), dict(exp_avgs=[b[:2]])):
        with pytest.raises(ValueError):
            vm.ClippedAdam([b], **kw)
    with pytest.raises(ValueError):
        vm.ClippedAdam([])


def test_scan_encoder_options():
    import videometamaterials_amd as vm
    for kw in (dict(cond_attention="none"), dict(cond_attention="self-stacked", cond_att_GRU=True), dict(cond_attention="self-stacked", per_frame_cond=True)):
        with pytest.raises(ValueError):
            vm.Unet3D(dim=16, cond_att_scan=True, **kw)
    plain = vm.Unet3D(dim=16, cond_attention="self-stacked")
    assert not [k for k in plain.state_dict() if "scan" in k]
    m = vm.Unet3D(dim=16, cond_attention="self-stacked", cond_attention_tokens=40, cond_att_scan=True)
    assert len([k for k in m.state_dict() if k.startswith("sign_emb_scan.")]) == 24
    assert [k for k in m.state_dict() if "scan" not in k] == list(plain.state_dict())
