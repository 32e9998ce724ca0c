"""Wait states behind matrix instructions, in the built library itself.

A vector, LDS or memory instruction may read (or overwrite) the result of a matrix instruction of P passes P + 3 wait states after it at the earliest (fp32 operands:
P + 2); nothing in the hardware waits.  (A later matrix instruction starts P wait states after it, whatever the code says: the unit takes one at a time.)  The compiler fills the distance with s_nop, but where a branch in between is jumped over it has counted the instructions
of the other way: what follows the shorter way then reads results that are not there yet, and differs from run to run.  So every way from every matrix instruction
is walked here, in the disassembly of what this package's sources were compiled to."""
import os
import re
import shutil
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "videometamaterials_amd")
LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
# passes of the dense forms on gfx950, by rows x columns x depth of 16-bit operands; fp32 ones below
PASSES = {"32x32x16": 8, "16x16x32": 4, "32x32x8": 8, "16x16x16": 4, "4x4x4": 2}
PASSES_F32 = {"32x32x2": 16, "16x16x4": 8, "32x32x1": 16, "16x16x1": 8, "4x4x1": 2}


def code_objects(library):
    """The gfx950 ELF images in a host library's .hip_fatbin section."""
    dump = library + ".fatbin.tmp"
    subprocess.run([os.path.join(LLVM, "llvm-objcopy"), "--dump-section", f".hip_fatbin={dump}", library, os.devnull], check=True)
    with open(dump, "rb") as f:
        data = f.read()
    os.remove(dump)
    at = data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(n):
            offset, size, name = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + name]:
                yield data[at + offset:at + offset + size]
            p += 24 + name
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 24)


def functions(text):
    """name -> [(address, opcode, operands)] of a disassembly."""
    found, current = {}, None
    for line in text.splitlines():
        if line[:1] == "\t":
            body, _, note = line.strip().partition("//")
            if current is not None and note:
                op, _, rest = body.strip().partition(" ")
                target = re.search(r"<[^>]*\+0x([0-9a-f]+)>", note)
                current.append((int(note.split(":")[0], 16), op, rest, int(target.group(1), 16) if target else 0))
        else:
            m = re.match(r"([0-9a-f]+) <(\S+)>:", line)
            if m:
                current = found.setdefault(m.group(2), [])
    return found


def registers(operands):
    """Vector registers that a list of operands names: VGPR n as n, AGPR n as 1000 + n."""
    out = set()
    for kind, one, low, high in re.findall(r"(?<![\w.])([va])(?:(\d+)|\[(\d+):(\d+)\])", operands):
        base = 1000 if kind == "a" else 0
        out.update([base + int(one)] if one else range(base + int(low), base + int(high) + 1))
    return out


def needed(op):
    """Passes of a matrix instruction, and wait states between it and what reads its result."""
    size = re.search(r"_(\d+x\d+x\d+)", op).group(1)
    if op.endswith("f32"):
        return PASSES_F32[size], PASSES_F32[size] + 2
    return PASSES[size], PASSES[size] + 3


def too_early(code):
    """(wait states, needed, address of the matrix instruction, of the reader) wherever one comes too early on some way through the function."""
    index = {address: i for i, (address, _, _, _) in enumerate(code)}
    start = code[0][0]
    regs = [registers(rest) if op[:2] in ("v_", "ds") or op.split("_")[0] in ("buffer", "global", "flat", "scratch") else frozenset() for _, op, rest, _ in code]

    def after(i):
        op = code[i][1]
        if op == "s_endpgm":
            return ()
        if op == "s_branch":
            return (index[start + code[i][3]],)
        if op.startswith("s_cbranch"):
            return (i + 1, index[start + code[i][3]])
        return (i + 1,) if i + 1 < len(code) else ()

    bad = []
    for i, (address, op, rest, _) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result, (passes, need), best = registers(re.split(r",\s*(?![^\[]*\])", rest)[0]), needed(op), {}
        ways = [(j, 0) for j in after(i)]
        while ways:
            j, waited = ways.pop()
            if waited >= need or best.get(j, need) <= waited:
                continue
            best[j] = waited
            _, o, r, _ = code[j]
            if o.startswith("v_mfma"):
                parts = re.split(r",\s*(?![^\[]*\])", r)
                if (registers(parts[1]) | registers(parts[2])) & result:
                    bad.append((waited, need, address, code[j][0]))
                    continue
                if result <= registers(parts[0]):  # the same sum goes on: its readers are those of that instruction
                    continue
                waited = max(waited, passes)
            elif regs[j] & result:
                bad.append((waited, need, address, code[j][0]))
                continue
            ways += [(k, waited + (int(r, 0) + 1 if o == "s_nop" else 1)) for k in after(j)]
    return bad


def test_the_walk_finds_the_shorter_way():
    """The check itself on three small programs: a branch over instructions that the distance was counted with, the same with the distance kept, a straight line."""
    product = (0, "v_mfma_f32_32x32x16_bf16", "v[0:15], v[20:23], v[24:27], v[0:15]", 0)
    read = "v_add_f32_e32", "v40, v3, v40", 0

    def program(*lines):
        return [(4 * k, *line) for k, line in enumerate(lines)]
    jump, other = ("s_cbranch_scc1", "3", 16), ("ds_read_b128", "v[30:33], v41", 0)
    assert too_early(program(product[1:], jump, other, ("s_nop", "9", 0), read)) == [(1, 11, 0, 16)]
    assert too_early(program(product[1:], jump, other, ("s_nop", "7", 0), ("s_nop", "9", 0), read)) == []
    assert too_early(program(product[1:], ("s_nop", "9", 0), read)) == [(10, 11, 0, 8)]
    assert too_early(program(product[1:], ("s_nop", "10", 0), read)) == []
    assert too_early(program(product[1:], ("v_mfma_f32_32x32x16_bf16", "v[50:65], v[20:23], v[24:27], v[50:65]", 0), ("s_nop", "1", 0), read)) == []


@pytest.mark.parametrize("name", ["libvmm_hip.so", "libvmm_hip_exp.so"])
def test_results_of_matrix_instructions_are_waited_for(name, tmp_path):
    library = os.path.join(PACKAGE, name)
    if not os.path.exists(library) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("not built here, or no disassembler")
    copy = shutil.copy(library, tmp_path / name)
    products, found = 0, []
    for n, image in enumerate(code_objects(str(copy))):
        path = tmp_path / f"{n}.elf"
        path.write_bytes(image)
        text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", str(path)], check=True, capture_output=True, text=True).stdout
        for function, code in functions(text).items():
            here = sum(op.startswith("v_mfma") for _, op, _, _ in code)
            products += here
            if here:
                found += [f"{function}: {w} of {need} wait states from {a:#x} to {b:#x}" for w, need, a, b in too_early(code)]
    assert products > 1000
    assert not found, "\n".join(found[:40])


def test_tiles_have_landed_at_every_barrier(tmp_path):
    """The product kernel of the gated feed-forward fetches its tiles to LDS directly, and other waves read them behind the next barrier: on every way from such a load
    to a barrier the wave has to wait for it (vmcnt(0)).  The barrier does not do that by itself."""
    library = os.path.join(PACKAGE, "libvmm_hip.so")
    if not os.path.exists(library) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("not built here, or no disassembler")
    copy = shutil.copy(library, tmp_path / "l.so")
    kernels = loads = 0
    for n, image in enumerate(code_objects(str(copy))):
        path = tmp_path / f"{n}.elf"
        path.write_bytes(image)
        if b"ff_gemm_kernel" not in image:
            continue
        text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", str(path)], check=True, capture_output=True, text=True).stdout
        for function, code in functions(text).items():
            if "ff_gemm_kernel" not in function or not code:
                continue
            kernels += 1
            index, start = {address: i for i, (address, _, _, _) in enumerate(code)}, code[0][0]
            for i, (address, op, rest, _) in enumerate(code):
                if not (op.startswith("buffer_load") and rest.endswith("lds")):
                    continue
                loads += 1
                seen, ways = set(), [i + 1]
                while ways:
                    j = ways.pop()
                    if j in seen or j >= len(code):
                        continue
                    seen.add(j)
                    _, o, r, target = code[j]
                    if o == "s_endpgm" or (o == "s_waitcnt" and "vmcnt(0)" in r):
                        continue
                    assert o != "s_barrier", f"{function}: {code[j][0]:#x} is reached with the load of {address:#x} under way"
                    if o == "s_branch" or o.startswith("s_cbranch"):
                        ways.append(index[start + target])
                    if o != "s_branch":
                        ways.append(j + 1)
    assert kernels == 18 and loads > 18 * 8
