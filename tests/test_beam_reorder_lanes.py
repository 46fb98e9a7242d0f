"""k_beam_reorder takes the beams' pages out of other lanes of a wavefront, in the assembly that hipcc makes of it (no GPU).
A lane of a thread without a piece to copy may hold a beam's page, so that all of them are read while every lane is on:
behind the branch that the idle ones leave by, a register that the compiler moved would hold it in the others only."""

import importlib.util
import re
import subprocess

import pytest

from conftest import ROOT

CSRC = ROOT / "esep-soup-kernels_amd" / "csrc"


@pytest.fixture(scope="module")
def asm():
    spec = importlib.util.spec_from_file_location("esep_build", CSRC.parent / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    res = subprocess.run([build.HIPCC, *build.CFLAGS, "--cuda-device-only", "-S", str(CSRC / "paged.hip"), "-o", "-"],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return res.stdout


@pytest.mark.parametrize("most", [4, 8, 16, 32])
def test_pages_are_read_before_lanes_are_switched_off(asm, most):
    kernel = asm[re.search(rf"^\S*k_beam_reorderILi{most}E\S*:", asm, re.M).end():]
    kernel = kernel[:kernel.index("s_endpgm")]
    assert kernel.count("ds_bpermute") == 1  # the parents' pages
    run = kernel[kernel.index("ds_bpermute"):]
    run = run[:re.search(r"\n\ts_\w*saveexec\w* |\n\ts_mov_b64 exec,", run).start()]
    lanes = {}
    for reg, lane in re.findall(r"v_readlane_b32 \w+, (v\d+), (\d+)", run):
        lanes.setdefault(reg, set()).add(int(lane))
    whole = [reg for reg, x in lanes.items() if x >= set(range(most))]
    assert len(whole) == 2, lanes  # the beams' own pages and their parents'
