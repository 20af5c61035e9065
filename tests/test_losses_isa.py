"""What the compiler makes of the decoder losses' kernels (gfx950 assembly, no GPU needed): the large tiles' K loops may
hold neither register spills nor waits of the compiler's own (each would drain the LDS-DMA stream that the schedule keeps
in flight), and no kernel of these operators may use packed fp32 arithmetic."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"
pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")


def _asm(source, tmp_path, f16=False):
    """the assembly that the Makefile's own command for this source gives"""
    out = tmp_path / (source + ".s")
    obj = source + ("_f16.o" if f16 else ".o")
    csrc = os.path.join(ROOT, "clip_amd", "csrc")
    cmd = subprocess.run(["make", "-n", "-B", obj], cwd=csrc, check=True, capture_output=True, text=True).stdout.strip().split("\n")[-1]
    args = cmd.replace(f"-o {obj}", f"-o {out}").replace(" -c ", " -S --cuda-device-only ").split()
    subprocess.run(args, cwd=csrc, check=True, capture_output=True, timeout=600)
    return out.read_text()


def _kernels(asm):
    for name in re.findall(r"amdhsa_kernel (\S+)", asm):
        start = re.search(r"^" + re.escape(name) + r":", asm, re.M).end()
        yield name, asm[start:asm.index(".amdhsa_kernel", start)].split("\n")


@pytest.mark.parametrize("f16", [False, True])
def test_k_loops_of_the_large_tiles(tmp_path, f16):
    asm = _asm("vocab8", tmp_path, f16)
    seen = 0
    for name, body in _kernels(asm):
        if "vocab8_kernel" not in name:
            continue
        seen += 1
        depth, deepest, inside = 0, 0, []
        for i, line in enumerate(body):
            m = re.match(r"^(?:\.LBB\S+:|; %bb\.\d+:)(.*)", line)
            if m:
                d = re.search(r"Depth=(\d+)", m.group(1))
                depth = int(d.group(1)) if d else depth if "Loop" in m.group(1) else 0
            inside.append(depth)
            if "v_mfma" in line:
                deepest = max(deepest, depth)
        assert deepest >= 1
        loop = [i for i, d in enumerate(inside) if d == deepest]
        assert sum("v_mfma" in body[i] for i in loop) >= 128
        assert not [body[i] for i in loop if "scratch_" in body[i]], name
        waits = [body[i].strip() for i in loop if "s_waitcnt" in body[i] and "vmcnt" in body[i] and "ASMSTART" not in body[i - 1]]
        assert not waits, (name, waits[:3])
    assert seen == 3


@pytest.mark.parametrize("source", ["vocab", "vocab8", "topk"])
def test_no_packed_fp32(tmp_path, source):
    asm = _asm(source, tmp_path)
    assert not re.findall(r"v_pk_(?:add|mul|fma)_f32", asm)
