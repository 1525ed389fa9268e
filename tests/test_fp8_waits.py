"""CPU: the module that the 8-bit products compile to.  Every read of the LDS behind a
wait for DMAs is kept there by the source, not by the order that a compiler happens to
choose; and no kernel is built that no call reaches.

The DMAs are inline assembly and the wait an intrinsic without memory effects, so a
plain read may move across it unless an assembly statement that clobbers memory
stands between them."""
import re
import shutil
import subprocess

import pytest

from zoomkv_revision_amd.build import CFLAGS, CSRC, HIPCC

pytestmark = pytest.mark.skipif(not shutil.which(HIPCC), reason="needs hipcc")


def unfenced(ir: str) -> list[str]:
    """Functions of an LLVM module in which a read of the LDS follows a vmcnt wait
    with no memory-clobbering assembly between."""
    bad = []
    for name, body in re.findall(r"^define [^\n]*@(\w+)\(.*?\{\n(.*?)^\}", ir, re.M | re.S):
        waited = False
        for line in body.splitlines():
            if "@llvm.amdgcn.s.waitcnt(" in line:
                waited = True
            elif "asm sideeffect" in line and "~{memory}" in line:
                waited = False
            elif waited and re.search(r"= load .*addrspace\(3\)", line):
                bad.append(name)
                break
    return bad


def test_a_read_without_its_fence_is_found():
    text = ("define void @k(i32 %%0) {\n  tail call void @llvm.amdgcn.s.waitcnt(i32 3952)\n%s"
            "  %%2 = load float, ptr addrspace(3) %%1, align 4\n}\n")
    assert unfenced(text % "") == ["k"]
    assert unfenced(text % "  tail call void asm sideeffect \"\", \"~{memory}\"() #1\n") == []


@pytest.fixture(scope="module")
def module(tmp_path_factory):
    out = tmp_path_factory.mktemp("ir") / "fp8_linear.ll"
    cmd = [HIPCC, *CFLAGS, "--cuda-device-only", "-emit-llvm", "-S", str(CSRC / "fp8_linear.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True)
    ir = out.read_text()
    return ir, set(re.findall(r"^define amdgpu_kernel [^\n]*@(\w+)\(", ir, re.M))


def test_reads_stay_behind_their_waits(module):
    ir, kernels = module
    assert sum("fp8_stream_kernel" in k for k in kernels) >= 6 and sum("fp8_tile_kernel" in k for k in kernels) == 5
    assert unfenced(ir) == []


def test_the_join_of_one_run_is_the_gated_one(module):
    """A linear product in one run leaves no sums; a gated one leaves its two parts'."""
    runs = lambda name: sorted(int(n) for k in module[1] for n in re.findall(name + r"ILi(\d+)E", k))
    assert runs("fp8_gated_join_kernel") == list(range(1, 9)) and runs("15fp8_join_kernel") == list(range(2, 9))
